// Linear layers with 4-bit weights and FP16 group scales, for the few tokens of a decode step:
//     y[m,n] = sum_g s[n,g] * sum_{k in g} x[m,k] q[n,k] + bias[n],   q in -8..7.
//
// Storage of q: a row's K values in blocks of 128 (64 bytes, the last padded with zeros), a block
// a 4 x 4 transpose of its 32-bit words: word 4 g + j holds values 32 j + 8 g .. + 7, so that the
// 16 bytes that lane group g of a wave loads are its operands of four 32-deep products in turn, each
// inside one scale group (32, 64 or 128 values). In a word, value 2 i lies at bits 4 i and value
// 2 i + 1 at bits 16 + 4 i (plus 8): a shift and a mask leave two neighbours in the two halves.
#include "float16_types.h"
#include "lds_dma.h"


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

// One thread per word; the threads of a scale group (4, 8 or 16) are neighbours. Bound: reading w once, value by value: 8192 x 11008
// 81 to 91 us, 2.8 TB/s from FP16, 4.5 to 4.9 from FP32 (packing 56, 2.4).
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

// Eight stored values as a product's operand, exact: q for FP16, q / 16 for BF16 (kUnit, which the group's scale takes
// back). FP16: nibble | 0x6400 is 1024 + nibble, and the exact packed subtraction of 1032 leaves q; the odd
// nibbles are taken in place, 1024 + 16 nibble, by an exact multiply-add (the published trick of 16-bit
// exponent bits under a small integer). BF16 has no packed arithmetic: the nibbles, made two's complement by their top
// bits, are converted to FP32 sixteenths one by one and packed in pairs, 14 instructions a word against FP16's 9 (us, FP16 /
// BF16: 1 token of 8192 x 11008 12.7 / 13.5, 16 tokens 13.9 / 15.7, 64 tokens 25.8 / 25.4). A shifted weight, 136 + q in 7
// instructions, would need -136 x beside it: sums 17 times as large, and inf - inf for an infinite x.
template <class T>
struct Int4Operand {
    static constexpr float kUnit = std::is_same<T, Fp16>::value ? 1.0f : 0.0625f;
    uint32_t top;   // FP16's exponent bits, in a register: and-or takes one constant from elsewhere
    __device__ __forceinline__ Int4Operand() : top(0x64006400u) { asm volatile("" : "+v"(top)); }
    __device__ __forceinline__ v4u operator()(uint32_t w) const {
        if constexpr (std::is_same<T, Fp16>::value) {
            const uint32_t hi = w >> 8;
            const Fp16::v2 sub = {-1032.0f16, -1032.0f16}, mul = {0.0625f16, 0.0625f16}, add = {-72.0f16, -72.0f16};
            auto even = [&](uint32_t b) {
                return __builtin_bit_cast(uint32_t, __builtin_bit_cast(Fp16::v2, (b & 0x000F000Fu) | top) + sub);
            };
            auto odd = [&](uint32_t b) {
                return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(
                                                        __builtin_bit_cast(Fp16::v2, (b & 0x00F000F0u) | top), mul, add));
            };
            return v4u{even(w), odd(w), even(hi), odd(hi)};
        } else {
            const uint32_t even = w ^ 0x88888888u;
            uint32_t odd = even >> 4;
            asm volatile("" : "+v"(odd));                            // so that the conversions select bytes of it
            auto at = [](uint32_t b, int shift) {
                return T::pack(__builtin_amdgcn_cvt_off_f32_i4(static_cast<int>(b >> shift & 255u)),
                               __builtin_amdgcn_cvt_off_f32_i4(static_cast<int>(b >> (16 + shift) & 255u)));
            };
            return v4u{at(even, 0), at(odd, 0), at(even, 8), at(odd, 8)};
        }
    }
};

struct Int4Args {
    const uint16_t* x;
    const uint8_t* w;
    const uint16_t* scale;
    const uint16_t* bias;
    uint16_t* out;
    int M, K, N;
};

// Rows shorter than a unit of 256 values: a thread per result.
template <class T>
__global__ __launch_bounds__(256) void int4_short_kernel(Int4Args a, int group)
{
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<long long>(a.M) * a.N) return;
    const int m = static_cast<int>(i / a.N), n = static_cast<int>(i - static_cast<long long>(m) * a.N);
    const int blocks = (a.K + kInt4Block - 1) / kInt4Block, groups = a.K / group;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(a.w + static_cast<size_t>(n) * blocks * 64);
    const uint16_t* x = a.x + static_cast<size_t>(m) * a.K;
    float acc = 0.0f;
    for (int k0 = 0; k0 < a.K; k0 += group) {
        float sum = 0.0f;
        for (int k = k0; k < k0 + group; k += 8) {
            const uint32_t q = w[int4_word_at(k / 8)];
#pragma unroll
            for (int e = 0; e < 8; e++)
                sum = __builtin_fmaf(T::widen(x[k + e]), static_cast<float>(static_cast<int>(q >> (4 * (e >> 1) + 16 * (e & 1)) & 15u) - 8), sum);
        }
        acc = __builtin_fmaf(sum, h2f(a.scale[static_cast<size_t>(n) * groups + k0 / group]), acc);
    }
    if (a.bias) acc += T::widen(a.bias[n]);
    a.out[i] = narrow<T>(acc);
}

// A workgroup computes 16 MT tokens x 16 NT rows; its W waves take the units of U (128 or 256) values
// of K in turn, each with the whole tile, and their FP32 sums are joined through LDS in wave order. Tokens
// are the A operand (rows), weight rows the B operand (columns): a lane's four accumulators are four tokens of one
// weight row, so a group's scale is one value per lane.
//
// Weights, scales and tokens come by LDS DMA into a ring of S units that each wave has for itself (no
// barrier while it streams): an operand's lanes lie 16 rows apart, and loaded as they lie each of the 64
// is a cache access of its own, 60 clocks an instruction whatever else was done (1 token 8192 x 11008 14 us, 64
// tokens 42). In LDS a row's 16-byte chunks are permuted so that 16 rows of one chunk fall on different
// banks. XR: rows of a token tile that are loaded (4 for up to 4 tokens, else 16; past M the last one again).
template <int U>
struct Int4Ring {
    static constexpr int kWChunks = U / 32, kXChunks = U / 8;        // 16-byte chunks of a row's unit
    static __device__ __forceinline__ int swz_w(int r) { return U == 256 ? (r >> 1) & 7 : (r >> 2) & 3; }
    static __device__ __forceinline__ int swz_x(int r) { return r & 15; }
};

template <class T, int G, int MT, int XR, int NT, int W, int U, int S>
__global__ __launch_bounds__(64 * W) void int4_linear_kernel(Int4Args a)
{
    using Ring = Int4Ring<U>;
    constexpr int kGroups = U / G, kBlocks = U / kInt4Block;         // of a unit
    constexpr int kWIns = kBlocks, kSIns = (16 * kGroups + 63) / 64, kXIns = XR * Ring::kXChunks / 64;
    constexpr int kIns = NT * (kWIns + kSIns) + MT * kXIns;          // DMA instructions of a unit
    constexpr int kS0 = NT * kWIns * 1024, kX0 = kS0 + NT * kSIns * 256, kStage = kX0 + MT * kXIns * 1024;
    constexpr int kSums = W * MT * NT * 1024, kLds = W * S * kStage > kSums ? W * S * kStage : kSums;
    static_assert(XR * Ring::kXChunks % 64 == 0 && kIns * (S - 1) < 64 && kLds <= 160 * 1024, "unit and ring sizes");
    __shared__ __align__(1024) int8_t lds[kLds];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int blocks = (a.K + kInt4Block - 1) / kInt4Block, units = (blocks + kBlocks - 1) / kBlocks, groups = a.K / G;

    // What lane l of each DMA instruction reads, as byte offsets from the tile's first row.
    const uint8_t* wbase = a.w + static_cast<size_t>(n0) * blocks * 64;
    const uint8_t* sbase = reinterpret_cast<const uint8_t*>(a.scale + static_cast<size_t>(n0) * groups);
    const uint8_t* xbase = reinterpret_cast<const uint8_t*>(a.x + static_cast<size_t>(m0) * a.K);
    uint32_t woff[NT][kWIns], soff[NT][kSIns], xoff[MT][kXIns];
    int wblk[kWIns], xk[kXIns];                                      // block and value of the unit
    const int sgrp = lane % kGroups;                                 // group
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < kWIns; i++) {
            const int c = i * 64 + lane, r = c / Ring::kWChunks, k = (c % Ring::kWChunks) ^ Ring::swz_w(r);
            woff[n][i] = static_cast<uint32_t>(min(16 * n + r, a.N - 1 - n0) * blocks * 64 + 16 * (k & 3));
            wblk[i] = k >> 2;
        }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < kSIns; i++)
            soff[n][i] = static_cast<uint32_t>(min(16 * n + ((i * 64 + lane) / kGroups & 15), a.N - 1 - n0) * groups * 2);
#pragma unroll
    for (int i = 0; i < kXIns; i++) {
        const int c = i * 64 + lane, r = c / Ring::kXChunks;
        xk[i] = 8 * ((c % Ring::kXChunks) ^ Ring::swz_x(r));
#pragma unroll
        for (int m = 0; m < MT; m++) xoff[m][i] = static_cast<uint32_t>(min(16 * m + r, a.M - 1 - m0) * a.K * 2);
    }
    const uint32_t mine = lds_address(lds) + wave * S * kStage;
    auto load = [&](int u, int slot) {
        const uint32_t to = mine + slot * kStage;
        const uint32_t sg = static_cast<uint32_t>(min(u * kGroups + sgrp, groups - 1)) * 2u;
#pragma unroll
        for (int i = 0; i < kWIns; i++) {
            const uint32_t b = static_cast<uint32_t>(min(u * kBlocks + wblk[i], blocks - 1)) * 64u;
#pragma unroll
            for (int n = 0; n < NT; n++) dma16_off(wbase, woff[n][i] + b, to + (n * kWIns + i) * 1024);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < kSIns; i++) dma2_off(sbase, soff[n][i] + sg, to + kS0 + (n * kSIns + i) * 256);
#pragma unroll
        for (int i = 0; i < kXIns; i++) {
            const uint32_t k = static_cast<uint32_t>(min(u * U + xk[i], a.K - 8)) * 2u;   // past K: not used
#pragma unroll
            for (int m = 0; m < MT; m++) dma16_off(xbase, xoff[m][i] + k, to + kX0 + (m * kXIns + i) * 1024);
        }
    };

    const int wr = col * Ring::kWChunks, xrow = col & (XR - 1), xr = xrow * Ring::kXChunks;
    const Int4Operand<T> operand;
    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) acc[m][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int count = wave < units ? (units - wave + W - 1) / W : 0;
#pragma unroll
    for (int i = 0; i < S; i++)
        if (i < count) load(wave + i * W, i);
    int slot = 0;
    for (int it = 0; it < count; it++) {
        if (it + S <= count) wait_vmcnt<kIns*(S - 1)>();
        else wait_vmcnt<0>();
        compiler_fence();
        const int u = wave + it * W;
        const int8_t* at = lds + (wave * S + slot) * kStage;
        v4f sum[MT][NT];
        float sc[NT][kGroups];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < kGroups; i++)
                sc[n][i] = h2f(*reinterpret_cast<const uint16_t*>(at + kS0 + n * kSIns * 256 + (col * kGroups + i) * 4)) *
                           (1.0f / Int4Operand<T>::kUnit);
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            v4u w[NT];
#pragma unroll
            for (int n = 0; n < NT; n++)
                w[n] = *reinterpret_cast<const v4u*>(at + n * kWIns * 1024 + (wr + ((4 * b + g) ^ Ring::swz_w(col))) * 16);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int step = 4 * b + j;                          // of 32 values
                const bool first = step % (G / 32) == 0, last = (step + 1) % (G / 32) == 0;
                const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
                v4u x[MT];
#pragma unroll
                for (int m = 0; m < MT; m++)
                    x[m] = *reinterpret_cast<const v4u*>(at + kX0 + m * kXIns * 1024 +
                                                         (xr + ((4 * step + g) ^ Ring::swz_x(xrow))) * 16);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const v4u q = operand(w[n][j]);
#pragma unroll
                    for (int m = 0; m < MT; m++) sum[m][n] = T::mfma16(x[m], q, first ? zero : sum[m][n]);
                }
                if (last && u * kGroups + step / (G / 32) < groups) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                acc[m][n][e] = __builtin_fmaf(sum[m][n][e], sc[n][step / (G / 32)], acc[m][n][e]);
                }
            }
        }
        if (it + S < count) {
            wait_lgkm0();                                            // the slot is read
            compiler_fence();
            load(u + S * W, slot);
        }
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    __syncthreads();
    v4f* part = reinterpret_cast<v4f*>(lds);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) part[(wave * MT * NT + m * NT + n) * kWave + lane] = acc[m][n];
    __syncthreads();
    // thread -> one output of the tile; its W partial sums in wave order
    const float* p = reinterpret_cast<const float*>(part);
    for (int i = threadIdx.x; i < MT * NT * 256; i += 64 * W) {
        const int n = i % (16 * NT), m = i / (16 * NT);
        if (m0 + m >= a.M || n0 + n >= a.N) continue;
        const int tile = (m / 16) * NT + n / 16;
        const int at = (tile * kWave + 16 * ((m % 16) / 4) + n % 16) * 4 + m % 4;
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < W; v++) s += p[v * (MT * NT * kWave * 4) + at];
        if (a.bias) s += T::widen(a.bias[n0 + n]);
        a.out[static_cast<size_t>(m0 + m) * a.N + n0 + n] = narrow<T>(s);
    }
}

template <class T, int G, int MT, int XR, int NT, int W, int U, int S>
int launch_int4(const Int4Args& a, hipStream_t s) {
    if (divup(a.N, 16 * NT) > grid_limit(64 * W)) return FORGE_EINVAL;
    const dim3 grid(static_cast<unsigned>(divup(a.N, 16 * NT)), static_cast<unsigned>(divup(a.M, 16 * MT)));
    int4_linear_kernel<T, G, MT, XR, NT, W, U, S><<<grid, 64 * W, 0, s>>>(a);
    return launch_status();
}

// 16 or 48 rows a workgroup: the one whose rounds over the CUs cost less, where a round of 48 rows takes
// `cost` percent of one of 16 (measured at K = 8192: the more tokens, the more of it is loading them).
inline bool int4_wide(int N, int cost) {
    const int cus = default_cu_count();
    return 100LL * divup(divup(N, 16), cus) > static_cast<long long>(cost) * divup(divup(N, 48), cus);
}

// us, 16 rows / 48 rows a workgroup: 16 tokens 4096 x 4096 4.3 / 7.4, 8192 x 11008 17.8 / 13.2; 32 tokens 5.5 / 9.0
// and 24.8 / 16.6; 64 tokens 8.1 / 12.8 and 41 / 25. Up to 4 tokens 16 waves stream 4096 x 4096 in 3.7 and 8192 x
// 11008 in 11.9 (47 MB, 4.1 TB/s; 4 waves 4.0 and 14); from 16384 rows on there are workgroups enough for 4
// waves each (2048 x 28000 7.9, 16 waves 9.9).
template <class T, int G>
int launch_int4(const Int4Args& a, hipStream_t s) {
    if (a.M <= 4)
        return a.N < 16384 ? launch_int4<T, G, 1, 4, 1, 16, 128, 2>(a, s) : launch_int4<T, G, 1, 4, 1, 4, 256, 2>(a, s);
    if (a.M <= 16)
        return int4_wide(a.N, 280) ? launch_int4<T, G, 1, 16, 3, 4, 128, 2>(a, s)
                                   : launch_int4<T, G, 1, 16, 1, 8, 256, 1>(a, s);
    if (a.M <= 32)
        return int4_wide(a.N, 200) ? launch_int4<T, G, 2, 16, 3, 8, 128, 1>(a, s)
                                   : launch_int4<T, G, 2, 16, 1, 8, 128, 1>(a, s);
    return int4_wide(a.N, 160) ? launch_int4<T, G, 4, 16, 3, 8, 128, 1>(a, s)
                               : launch_int4<T, G, 4, 16, 1, 8, 128, 1>(a, s);
}

template <class T>
int launch_int4(const Int4Args& a, int group, hipStream_t s) {
    if (a.K < 256) {
        const long long wgs = divupll(static_cast<long long>(a.M) * a.N, 256);
        if (wgs > grid_limit(256)) return FORGE_EINVAL;
        int4_short_kernel<T><<<static_cast<unsigned>(wgs), 256, 0, s>>>(a, group);
        return launch_status();
    }
    if (group == 32) return launch_int4<T, 32>(a, s);
    if (group == 64) return launch_int4<T, 64>(a, s);
    return launch_int4<T, 128>(a, s);
}

}  // namespace forge_amd

using namespace forge_amd;

namespace {
// (K: a tile's rows are addressed in 32 bits)
bool int4_shape_ok(int K, int group) { return (group == 32 || group == 64 || group == 128) && K % group == 0 && K <= 1 << 23; }
}  // namespace

extern "C" int forge_quantize_weight_int4(const void* w, int w_fp16, uint8_t* w_int4, uint16_t* w_scale, int N, int K,
                                          int group, void* stream)
{
    if (N <= 0 || K <= 0) return FORGE_OK;
    if (!w || !w_int4 || !w_scale || !aligned(w_int4, 16) || !int4_shape_ok(K, group)) return FORGE_EINVAL;
    const int row_words = int4_row_bytes(K) / 4;
    const long long words = static_cast<long long>(N) * row_words, wgs = divupll(words, 256);
    if (wgs > grid_limit(256)) return FORGE_EINVAL;
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
    if (wgs > grid_limit(256)) return FORGE_EINVAL;
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
