// Linear layers with 4-bit weights and FP16 group scales, for the few tokens of a decode step:
//     y[m,n] = sum_g s[n,g] * sum_{k in g} x[m,k] q[n,k] + bias[n],   q in -8..7.
//
// Storage of q: a row's K values in blocks of 128 (64 bytes, the last padded with zeros), a block
// a 4 x 4 transpose of its 32-bit words: word 4 g + j holds values 32 j + 8 g .. + 7, so that the
// 16 bytes that lane group g of a wave loads are its operands of four 32-deep products in turn, each
// inside one scale group (32, 64 or 128 values). In a word, value 2 i lies at bits 4 i and value
// 2 i + 1 at bits 16 + 4 i (plus 8): a shift and a mask leave two neighbours in the two halves.
#include "float16_types.h"
#include "mfma_tile.h"

#include <climits>

namespace forge_amd {

constexpr int kInt4Block = 128;

inline int int4_row_bytes(int K) { return divup(K, kInt4Block) * (kInt4Block / 2); }

// ---- weight preparation ---------------------------------------------------------------------------

// Eight integers -8..7 as one word of the storage.
__device__ __forceinline__ uint32_t int4_word(const int (&q)[8]) {
    uint32_t w = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) w |= static_cast<uint32_t>(q[e] + 8) << (4 * (e >> 1) + 16 * (e & 1));
    return w;
}
// Position of natural word c (values 8 c .. + 7) in its row.
__device__ __forceinline__ size_t int4_word_at(int c) {
    return static_cast<size_t>(c >> 4) * 16 + 4 * (c & 3) + ((c & 15) >> 2);
}

// One thread per word; the threads of a scale group (4, 8 or 16) are neighbours. Bound: reading w once.
template <bool FP16W>
__global__ __launch_bounds__(256) void quantize_weight_int4_kernel(const void* __restrict__ w, uint32_t* __restrict__ out,
                                                                   uint16_t* __restrict__ scale, int K, int group,
                                                                   long long words, int row_words)
{
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const long long n = i / row_words;
    const int c = static_cast<int>(i - n * row_words), k = 8 * c;
    const bool in = i < words && k < K;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    if (in) {
        const size_t at = static_cast<size_t>(n) * K + k;
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = FP16W ? h2f(static_cast<const uint16_t*>(w)[at + e]) : static_cast<const float*>(w)[at + e];
    }
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(v[e]));
    for (int d = 1; d < group / 8; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d, kWave));
    if (i >= words) return;
    // The stored FP16 scale divides, so that q is the nearest to w / scale as it will be used; a group too
    // small for FP16 takes the smallest positive scale.
    uint16_t s = f2h(amax / 7.0f);
    s = s ? s : uint16_t{1};
    const float sf = h2f(s);
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float r = __builtin_rintf(v[e] / sf);
        q[e] = (r == r) ? static_cast<int>(fminf(fmaxf(r, -8.0f), 7.0f)) : 0;
    }
    out[static_cast<size_t>(n) * row_words + int4_word_at(c)] = int4_word(q);
    if (in && k % group == 0) scale[static_cast<size_t>(n) * (K / group) + k / group] = s;
}

__global__ __launch_bounds__(256) void pack_weight_int4_kernel(const int8_t* __restrict__ w, uint32_t* __restrict__ out,
                                                               int K, long long words, int row_words)
{
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= words) return;
    const long long n = i / row_words;
    const int c = static_cast<int>(i - n * row_words), k = 8 * c;
    int q[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        q[e] = k < K ? min(max(static_cast<int>(w[static_cast<size_t>(n) * K + k + e]), -8), 7) : 0;
    out[static_cast<size_t>(n) * row_words + int4_word_at(c)] = int4_word(q);
}

// ---- the product -----------------------------------------------------------------------------------

// Eight stored values as a product's operand. FP16: nibble | 0x6400 is 1024 + nibble, and the exact
// packed subtraction of 1032 leaves q; the odd nibbles are taken in place, 1024 + 16 nibble, by an
// exact multiply-add. BF16 has no packed subtraction: nibble | 0x4300 is 128 + nibble = 136 + q, and
// the caller starts its sum from -136 x.
template <class T>
__device__ __forceinline__ v4u int4_operand(uint32_t w) {
    if constexpr (std::is_same<T, Fp16>::value) {
        const uint32_t hi = w >> 8;
        const Fp16::v2 sub = {-1032.0f16, -1032.0f16}, mul = {0.0625f16, 0.0625f16}, add = {-72.0f16, -72.0f16};
        auto even = [&](uint32_t b) {
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(Fp16::v2, (b & 0x000F000Fu) | 0x64006400u) + sub);
        };
        auto odd = [&](uint32_t b) {
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
                                                    __builtin_bit_cast(Fp16::v2, (b & 0x00F000F0u) | 0x64006400u), mul, add));
        };
        return v4u{even(w), odd(w), even(hi), odd(hi)};
    } else {
        auto at = [&](uint32_t b) { return (b & 0x000F000Fu) | 0x43004300u; };
        return v4u{at(w), at(w >> 4), at(w >> 8), at(w >> 12)};
    }
}

struct Int4Args {
    const uint16_t* x;
    const uint8_t* w;
    const uint16_t* scale;
    const uint16_t* bias;
    uint16_t* out;
    int M, K, N;
};

// A workgroup computes 16 MT tokens x 16 NT rows; its W waves take the 256-value units of K in
// turn, each with the whole tile, and their FP32 sums are joined through LDS in wave order. Tokens
// are the A operand (rows), weight rows the B operand (columns): a lane's four accumulators are four
// tokens of one weight row, so a group's scale is one value per lane.
template <class T, int G, int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void int4_linear_kernel(Int4Args a)
{
    __shared__ v4f part[W][MT * NT][kWave];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int blocks = (a.K + kInt4Block - 1) / kInt4Block;
    const int groups = a.K / G;

    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    const uint8_t* wrow[NT];
    const uint16_t* srow[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const size_t r = static_cast<size_t>(min(n0 + 16 * n + col, a.N - 1));
        wrow[n] = a.w + r * (static_cast<size_t>(blocks) * 64) + 16 * g;
        srow[n] = a.scale + r * groups;
    }
    const uint16_t* xrow[MT];
    bool live[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int r = m0 + 16 * m + col;
        live[m] = r < a.M;
        xrow[m] = a.x + static_cast<size_t>(live[m] ? r : 0) * a.K + 8 * g;
    }

    for (int b = wave; b < blocks; b += W) {
        v4u w[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) w[n] = *reinterpret_cast<const v4u*>(wrow[n] + static_cast<size_t>(b) * 64);
#pragma unroll
        for (int j0 = 0; j0 < 4; j0 += G / 32) {
            const int k0 = b * kInt4Block + 32 * j0;
            if (k0 >= a.K) break;
            v4f sum[MT][NT];
            v4f base[MT];
            v4u x[MT][G / 32];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                base[m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < G / 32; j++) {
                    x[m][j] = v4u{0u, 0u, 0u, 0u};
                    if (live[m]) x[m][j] = *reinterpret_cast<const v4u*>(xrow[m] + k0 + 32 * j);
                    if constexpr (std::is_same<T, Bf16>::value) {
                        const v4u c = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};   // -136
                        base[m] = T::mfma16(x[m][j], c, base[m]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float s = h2f(srow[n][k0 / G]);
#pragma unroll
                for (int m = 0; m < MT; m++) sum[m][n] = base[m];
#pragma unroll
                for (int j = 0; j < G / 32; j++) {
                    const v4u q = int4_operand<T>(w[n][j0 + j]);
#pragma unroll
                    for (int m = 0; m < MT; m++) sum[m][n] = T::mfma16(x[m][j], q, sum[m][n]);
                }
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[m][n][e] = __builtin_fmaf(sum[m][n][e], s, acc[m][n][e]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) part[wave][m * NT + n][lane] = acc[m][n];
    __syncthreads();
    // thread -> one output of the tile; its W partial sums in wave order
    const float* p = reinterpret_cast<const float*>(part);
    for (int i = threadIdx.x; i < MT * NT * 256; i += 64 * W) {
        const int n = i % (16 * NT), m = i / (16 * NT);
        const int tile = (m / 16) * NT + n / 16;
        const int at = (tile * kWave + 16 * ((m % 16) / 4) + n % 16) * 4 + m % 4;
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < W; v++) s += p[v * (MT * NT * kWave * 4) + at];
        if (m0 + m < a.M && n0 + n < a.N) {
            if (a.bias) s += T::widen(a.bias[n0 + n]);
            a.out[static_cast<size_t>(m0 + m) * a.N + n0 + n] = narrow<T>(s);
        }
    }
}

template <class T, int G>
int launch_int4(const Int4Args& a, hipStream_t s) {
    constexpr int NT = 1, W = 8;
    auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        const dim3 grid(static_cast<unsigned>(divup(a.N, 16 * NT)), static_cast<unsigned>(divup(a.M, 16 * MT)));
        int4_linear_kernel<T, G, MT, NT, W><<<grid, 64 * W, 0, s>>>(a);
        return launch_status();
    };
    if (a.M <= 16) return go(std::integral_constant<int, 1>());
    if (a.M <= 32) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 4>());
}

template <class T>
int launch_int4(const Int4Args& a, int group, hipStream_t s) {
    if (group == 32) return launch_int4<T, 32>(a, s);
    if (group == 64) return launch_int4<T, 64>(a, s);
    return launch_int4<T, 128>(a, s);
}

}  // namespace forge_amd

using namespace forge_amd;

namespace {
bool int4_shape_ok(int K, int group) { return (group == 32 || group == 64 || group == 128) && K % group == 0; }
}  // namespace

extern "C" int forge_quantize_weight_int4(const void* w, int w_fp16, uint8_t* w_int4, uint16_t* w_scale, int N, int K,
                                          int group, void* stream)
{
    if (N <= 0 || K <= 0) return FORGE_OK;
    if (!w || !w_int4 || !w_scale || !aligned(w_int4, 16) || !int4_shape_ok(K, group)) return FORGE_EINVAL;
    const int row_words = int4_row_bytes(K) / 4;
    const long long words = static_cast<long long>(N) * row_words, wgs = divupll(words, 256);
    if (wgs > INT_MAX) return FORGE_EINVAL;
    hipStream_t s = as_stream(stream);
    if (w_fp16)
        quantize_weight_int4_kernel<true><<<static_cast<unsigned>(wgs), 256, 0, s>>>(
            w, reinterpret_cast<uint32_t*>(w_int4), w_scale, K, group, words, row_words);
    else
        quantize_weight_int4_kernel<false><<<static_cast<unsigned>(wgs), 256, 0, s>>>(
            w, reinterpret_cast<uint32_t*>(w_int4), w_scale, K, group, words, row_words);
    return launch_status();
}

extern "C" int forge_pack_weight_int4(const int8_t* q, uint8_t* w_int4, int N, int K, void* stream)
{
    if (N <= 0 || K <= 0) return FORGE_OK;
    if (!q || !w_int4 || !aligned(w_int4, 16) || K % 32 != 0) return FORGE_EINVAL;
    const int row_words = int4_row_bytes(K) / 4;
    const long long words = static_cast<long long>(N) * row_words, wgs = divupll(words, 256);
    if (wgs > INT_MAX) return FORGE_EINVAL;
    pack_weight_int4_kernel<<<static_cast<unsigned>(wgs), 256, 0, as_stream(stream)>>>(
        q, reinterpret_cast<uint32_t*>(w_int4), K, words, row_words);
    return launch_status();
}

extern "C" int forge_int4_linear(const uint16_t* x, const uint8_t* w_int4, const uint16_t* w_scale, const uint16_t* bias,
                                 uint16_t* out, int M, int K, int N, int group, int dtype, void* stream)
{
    if (M <= 0 || K <= 0 || N <= 0) return FORGE_OK;
    if (!x || !w_int4 || !w_scale || !out || !aligned(x, 16) || !aligned(w_int4, 16) || !int4_shape_ok(K, group) ||
        (dtype != FORGE_FP16 && dtype != FORGE_BF16) || divup(M, 64) > 65535)
        return FORGE_EINVAL;
    const Int4Args a{x, w_int4, w_scale, bias, out, M, K, N};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_int4<Fp16>(a, group, s) : launch_int4<Bf16>(a, group, s);
}
