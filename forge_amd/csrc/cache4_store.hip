// Keys and values into the 4-bit cache, and back into 16 bits.
//
// Per head: m = min x, s = (max / 15 - min / 15 in FP32) rounded toward zero to the 16-bit type, so that no m + s n
// passes its largest value, and n = round_half_even((x - m) / s), at most 15 (0 where s is 0). A head that holds an infinity or NaN has none of
// that: its s and m are NaN, and so is what reads it. Read: m + s n in FP32, rounded once.
// Bound: memory; a lane has a word of 8 values of a key and its value, a workgroup one head of 8, 16 or 32 neighbouring tokens, whose words and
// numbers then make whole cache lines. 16384 tokens of 8 heads of 128: written in 21.6 us (67 MB read of 20 KB rows, 18 MB written; 320 vector instructions a
// wave are most of it), read in 14.9.
#include "cache4.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr long long kMaxStride = 1 << 25;   // elements; 32 tokens of them stay in 32 bits

struct Store4Args {
    const uint16_t *k, *v;
    uint16_t *k_out, *v_out;
    uint8_t* cache;
    const int32_t* slots;
    long long k_head, v_head, rows;
    size_t page_bytes;
    Cache4Layout at;
    int k_token, v_token;
    int T, D;
};

// x >= 0 rounded toward zero to 16 bits.
template <class T>
__device__ __forceinline__ uint16_t toward_zero(float x) {
    const uint16_t h = narrow<T>(x);
    return T::widen(h) > x ? static_cast<uint16_t>(h - 1) : h;
}

// The cache's row of token t, or -1. (Loaded for any t, so that no branch waits for it.)
__device__ __forceinline__ int store4_slot(const Store4Args& a, int t) {
    const int s = a.slots[min(t, a.T - 1)];
    return t < a.T && s < a.rows ? s : -1;
}
// The piece of a slot's page and head hk (of the whole workgroup).
__device__ __forceinline__ uint8_t* store4_piece(const Store4Args& a, int slot, int hk) {
    return a.cache + hk * a.at.piece() + static_cast<uint32_t>(slot >> a.at.page_shift) * a.page_bytes;
}

// Pairs of 16-bit numbers as integers of the same order, and back.
typedef short v2s __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2s ordered(v2s x) { return x ^ ((x >> 15) & static_cast<short>(0x7FFF)); }

// Least and largest value over the LPH lanes of a head, both of which are numbers of the type: as a pair, the least one negated, in registers
// (neighbours, pairs, then mirrored halves of 8 and 16 lanes).
template <int CTRL>
__device__ __forceinline__ v2s with_lane(v2s x) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false);
    return __builtin_elementwise_max(x, __builtin_bit_cast(v2s, y));
}
template <class T, int LPH>
__device__ __forceinline__ void head_range(float* low, float* top) {
    v2s x = ordered(__builtin_bit_cast(v2s, T::pack(*top, -*low)));
    x = with_lane<0xB1>(x);
    x = with_lane<0x4E>(x);
    x = with_lane<0x141>(x);
    if (LPH >= 16) x = with_lane<0x140>(x);
    if (LPH >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const v2u r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t r0 = r[0], r1 = r[1];                         // (a bit cast of r[1] itself takes r[0])
        x = __builtin_elementwise_max(__builtin_bit_cast(v2s, r0), __builtin_bit_cast(v2s, r1));
    }
    x = ordered(x);
    *top = T::widen(static_cast<uint16_t>(x[0]));
    *low = -T::widen(static_cast<uint16_t>(x[1]));
}

// x / 15, correctly rounded: the product with the rounded reciprocal, corrected by its exact remainder, which FP32 holds for FP16's values.
template <class T>
__device__ __forceinline__ float fifteenth(float x) {
    if constexpr (T::kWide) return x / 15.0f;
    constexpr float kInv = 1.0f / 15.0f;
    const float q = x * kInv;
    return __builtin_fmaf(__builtin_fmaf(-15.0f, q, x), kInv, q);
}

// A head's 8 values of this lane: its word, and (on all lanes) step and lowest value.
template <class T, int LPH>
__device__ __forceinline__ uint32_t quantize_head(v4u own, bool in, uint32_t* numbers) {
    float x[8];
    widen8<T>(own, x);
    float low = INFINITY, top = -INFINITY;
    float odd = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        low = fminf(low, x[e]);
        top = fmaxf(top, x[e]);
    }
#pragma unroll
    for (int d = 0; d < 4; d++) odd = T::times_zero(own[d], odd);
    top = odd != 0.0f ? INFINITY : top;                              // an infinity or NaN
    low = in ? low : INFINITY;
    top = in ? top : -INFINITY;
    head_range<T, LPH>(&low, &top);
    constexpr uint32_t kNaN = T::kInfinity | T::kInfinity >> 1;
    *numbers = kNaN | kNaN << 16;
    if (!(top < INFINITY)) return 0u;
    const uint16_t step = toward_zero<T>(fifteenth<T>(top) - fifteenth<T>(low));
    *numbers = step | static_cast<uint32_t>(narrow<T>(low)) << 16;
    const float s = T::widen(step) * 0.5f, m = low * 0.5f;           // halves: x - m stays in range
    if (!in || !(s > 0.0f)) return 0u;
    // A product with the reciprocal is the quotient but for 2^-21 of it; only next to a half (or with a subnormal step) does it take
    // the division to know where that rounds. kWhole's sum with a small number rounds it to an integer in its last bits. 16384 tokens of
    // 8 heads of 128: eight divisions a lane 29 us, this 22.
    constexpr float kWhole = 12582912.0f;
    constexpr uint32_t kBits = 0x4B400000u;
    const float inv = __builtin_amdgcn_rcpf(s);
    // (A step of all its bits takes no quotient to 15.5.)
    float n[8], off = s < T::kNormal ? 1.0f : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float q = x[e] * 0.5f - m;
        n[e] = __builtin_fmaf(q, inv, kWhole);
        off = fmaxf(off, fabsf(__builtin_fmaf(q, inv, kWhole - n[e])));
    }
    if (__any(!(off < 0.49999f))) {
        asm volatile("" : "+v"(n[0]));                               // (the compiler would divide in any case)
#pragma unroll
        for (int e = 0; e < 8; e++) n[e] = fminf((x[e] * 0.5f - m) / s, 15.0f) + kWhole;
    }
    uint32_t word = 0u, all = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int shift = 4 * (e >> 1) + 16 * (e & 1);
        word += __float_as_uint(n[e]) << shift;
        all += kBits << shift;
    }
    return word - all;
}

template <class T, int LPH>
__global__ __launch_bounds__(256) void cache4_write_kernel(Store4Args a)
{
    const int lane = threadIdx.x & (kWave - 1), lh = lane & (LPH - 1), d0 = 8 * lh;
    const unsigned part = blockIdx.x / static_cast<unsigned>(a.at.Hkv);
    const int hk = blockIdx.x - part * a.at.Hkv, t = (part * 4 + threadIdx.x / kWave) * (kWave / LPH) + lane / LPH;
    const bool in = t < a.T && d0 < a.D;
    // (from the wave's first token on in 32 bits)
    const int t0 = __builtin_amdgcn_readfirstlane(t - lane / LPH), tt = min(lane / LPH, a.T - 1 - t0), dd = min(d0, a.D - 8);
    const v4u k = *reinterpret_cast<const v4u*>(a.k + static_cast<long long>(t0) * a.k_token + hk * a.k_head + (tt * a.k_token + dd));
    const v4u v = *reinterpret_cast<const v4u*>(a.v + static_cast<long long>(t0) * a.v_token + hk * a.v_head + (tt * a.v_token + dd));
    const int slot = store4_slot(a, t);
    v2u numbers;
    uint32_t kn, vn;
    const uint32_t kw = quantize_head<T, LPH>(k, in, &kn), vw = quantize_head<T, LPH>(v, in, &vn);
    numbers = v2u{kn, vn};
    if (slot < 0 || lh >= 4 * a.at.U) return;
    const int r = slot & ((1 << a.at.page_shift) - 1);
    uint8_t* piece = store4_piece(a, slot, hk);
    *reinterpret_cast<uint32_t*>(piece + a.at.key_row(r) + 4 * lh) = kw;
    *reinterpret_cast<uint32_t*>(piece + a.at.value_word(r, lh)) = vw;
    if (lh == 0) *reinterpret_cast<v2u*>(piece + a.at.numbers(r)) = numbers;
}

template <class T>
__device__ __forceinline__ v4u values_of(uint32_t word, uint32_t numbers) {
    const float s = T::widen(static_cast<uint16_t>(numbers & 0xFFFFu)), m = T::widen(static_cast<uint16_t>(numbers >> 16));
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(static_cast<float>(word >> (4 * (e >> 1) + 16 * (e & 1)) & 15u), s, m);
    return narrow8<T>(x);
}

template <class T, int LPH>
__global__ __launch_bounds__(256) void cache4_read_kernel(Store4Args a)
{
    const int lane = threadIdx.x & (kWave - 1), lh = lane & (LPH - 1), d0 = 8 * lh;
    const unsigned part = blockIdx.x / static_cast<unsigned>(a.at.Hkv);
    const int hk = blockIdx.x - part * a.at.Hkv, t = (part * 4 + threadIdx.x / kWave) * (kWave / LPH) + lane / LPH;
    if (t >= a.T || d0 >= a.D) return;
    const int slot = store4_slot(a, t);
    uint32_t kw = 0u, vw = 0u;                                       // a slot outside the cache: zeros
    v2u numbers = {0u, 0u};
    if (slot >= 0) {
        const int r = slot & ((1 << a.at.page_shift) - 1);
        const uint8_t* piece = store4_piece(a, slot, hk);
        kw = *reinterpret_cast<const uint32_t*>(piece + a.at.key_row(r) + 4 * lh);
        vw = *reinterpret_cast<const uint32_t*>(piece + a.at.value_word(r, lh));
        numbers = *reinterpret_cast<const v2u*>(piece + a.at.numbers(r));
    }
    const size_t out = (static_cast<size_t>(t) * a.at.Hkv + hk) * a.D + d0;
    *reinterpret_cast<v4u*>(a.k_out + out) = values_of<T>(kw, numbers[0]);
    *reinterpret_cast<v4u*>(a.v_out + out) = values_of<T>(vw, numbers[1]);
}

template <class T, int LPH>
int launch_store4(Store4Args a, bool write, hipStream_t s) {
    // as many tokens at a time as a grid holds
    constexpr int kTokens = 4 * kWave / LPH;                         // of a workgroup
    const int total = a.T;
    const long long most = grid_limit(256) / a.at.Hkv * kTokens;
    for (long long t = 0; t < total; t += most) {
        a.T = static_cast<int>(std::min(most, total - t));
        const unsigned grid = static_cast<unsigned>(divup(a.T, kTokens)) * a.at.Hkv;
        if (write) cache4_write_kernel<T, LPH><<<grid, 256, 0, s>>>(a);
        else cache4_read_kernel<T, LPH><<<grid, 256, 0, s>>>(a);
        const int st = launch_status();
        if (st != FORGE_OK) return st;
        a.slots += a.T;
        if (write) {
            a.k += static_cast<long long>(a.T) * a.k_token;
            a.v += static_cast<long long>(a.T) * a.v_token;
        } else {
            a.k_out += static_cast<size_t>(a.T) * a.at.Hkv * a.D;
            a.v_out += static_cast<size_t>(a.T) * a.at.Hkv * a.D;
        }
    }
    return FORGE_OK;
}

template <class T>
int launch_store4(const Store4Args& a, bool write, hipStream_t s) {
    if (a.D <= 64) return launch_store4<T, 8>(a, write, s);
    if (a.D <= 128) return launch_store4<T, 16>(a, write, s);
    return launch_store4<T, 32>(a, write, s);
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" int forge_cache4_write(const uint16_t* k, const uint16_t* v, uint8_t* cache, const int32_t* slots, int T, int Hkv,
                                  int D, int pages, int page_size, long long k_token, long long k_head, long long v_token,
                                  long long v_head, int dtype, void* stream)
{
    if (T <= 0 || Hkv <= 0 || D <= 0) return FORGE_OK;
    if (!cache4_shape_ok(Hkv, D, pages, page_size) || T > INT_MAX - 64 || !k || !v || !cache || !slots || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(cache)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    for (long long st : {k_token, k_head, v_token, v_head})
        if (st < 0 || st % 8 != 0 || st > kMaxStride) return FORGE_EINVAL;
    const Cache4Layout at{cache4_units(D), __builtin_ctz(static_cast<unsigned>(page_size)), Hkv};
    const Store4Args a{k, v, nullptr, nullptr, cache, slots, k_head, v_head, static_cast<long long>(pages) * page_size, at.at(1, 0), at,
                       static_cast<int>(k_token), static_cast<int>(v_token), T, D};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_store4<Fp16>(a, true, s) : launch_store4<Bf16>(a, true, s);
}

extern "C" int forge_cache4_read(const uint8_t* cache, const int32_t* slots, uint16_t* k, uint16_t* v, int T, int Hkv, int D,
                                 int pages, int page_size, int dtype, void* stream)
{
    if (T <= 0 || Hkv <= 0 || D <= 0) return FORGE_OK;
    if (!cache4_shape_ok(Hkv, D, pages, page_size) || T > INT_MAX - 64 || !k || !v || !cache || !slots || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(cache)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    const Cache4Layout at{cache4_units(D), __builtin_ctz(static_cast<unsigned>(page_size)), Hkv};
    const Store4Args a{nullptr, nullptr, k, v, const_cast<uint8_t*>(cache), slots, 0, 0, static_cast<long long>(pages) * page_size,
                       at.at(1, 0), at, 0, 0, T, D};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_store4<Fp16>(a, false, s) : launch_store4<Bf16>(a, false, s);
}
