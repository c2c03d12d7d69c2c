// Keys and values into the 4-bit cache, and back into 16 bits.
//
// Per head: m = min x, s = (max / 15 - min / 15 in FP32) rounded toward zero to the 16-bit type, so that no m + s n
// passes its largest value, and n = round_half_even((x - m) / s), at most 15 (0 where s is 0). A head that holds an infinity or NaN has none of
// that: its s and m are NaN, and so is what reads it. Read: m + s n in FP32, rounded once.
// Bound: memory; a lane has a word of 8 values, a wave one head of some neighbouring tokens, whose words of the values
// (4 bytes every 16) then make whole cache lines.
#include "cache4.h"

#include <algorithm>

namespace forge_amd {

struct Store4Args {
    const uint16_t *k, *v;
    uint16_t *k_out, *v_out;
    uint8_t* cache;
    const int32_t* slots;
    long long k_token, k_head, v_token, v_head, rows;
    Cache4Layout at;
    int T, D;
};

// x >= 0 rounded toward zero to 16 bits.
template <class T>
__device__ __forceinline__ uint16_t toward_zero(float x) {
    const uint16_t h = narrow<T>(x);
    return T::widen(h) > x ? static_cast<uint16_t>(h - 1) : h;
}

// The cache's row of token t, or -1.
__device__ __forceinline__ long long store4_slot(const Store4Args& a, int t) {
    const long long s = t < a.T ? a.slots[t] : -1;
    return s < a.rows ? s : -1;
}

template <class T, int LPH>
__global__ __launch_bounds__(256) void cache4_write_kernel(Store4Args a)
{
    const int lane = threadIdx.x & (kWave - 1), lh = lane & (LPH - 1), d0 = 8 * lh;
    const int t = blockIdx.x * (kWave / LPH) + lane / LPH;
    const int h = blockIdx.y * 4 + threadIdx.x / kWave;              // keys' heads, then values'
    if (h >= 2 * a.at.Hkv) return;
    const bool is_v = h >= a.at.Hkv;
    const int hk = is_v ? h - a.at.Hkv : h;
    const long long slot = store4_slot(a, t);
    const bool in = slot >= 0 && d0 < a.D;
    v4u own = {0u, 0u, 0u, 0u};
    if (in) own = *reinterpret_cast<const v4u*>((is_v ? a.v + t * a.v_token + hk * a.v_head : a.k + t * a.k_token + hk * a.k_head) + d0);
    float x[8];
    widen8<T>(own, x);
    float low = INFINITY, top = -INFINITY, odd = 0.0f;
    if (in) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            low = fminf(low, x[e]);
            top = fmaxf(top, x[e]);
        }
#pragma unroll
        for (int d = 0; d < 4; d++) odd = T::times_zero(own[d], odd);
    }
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) {
        low = fminf(low, __shfl_xor(low, o, kWave));
        top = fmaxf(top, __shfl_xor(top, o, kWave));
        odd += __shfl_xor(odd, o, kWave);
    }
    if (slot < 0 || lh >= 4 * a.at.U) return;
    const uint16_t step = toward_zero<T>(top / 15.0f - low / 15.0f);
    const float s = T::widen(step) * 0.5f, m = low * 0.5f;           // halves: x - m stays in range
    uint32_t word = 0u;
    if (d0 < a.D && odd == 0.0f && s > 0.0f) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float n = fminf(__builtin_rintf((x[e] * 0.5f - m) / s), 15.0f);
            word |= static_cast<uint32_t>(n) << (4 * (e >> 1) + 16 * (e & 1));
        }
    }
    const int r = static_cast<int>(slot) & ((1 << a.at.page_shift) - 1);
    uint8_t* piece = a.cache + a.at.at(slot >> a.at.page_shift, hk);
    *reinterpret_cast<uint32_t*>(piece + (is_v ? a.at.value_word(r, lh) : a.at.key_row(r) + 4 * lh)) = word;
    if (lh == 0) {
        const uint32_t nan = T::kInfinity | T::kInfinity >> 1;       // a quiet NaN
        const uint32_t numbers = odd == 0.0f ? step | static_cast<uint32_t>(narrow<T>(low)) << 16 : nan | nan << 16;
        *reinterpret_cast<uint32_t*>(piece + a.at.numbers(r) + (is_v ? 4 : 0)) = numbers;
    }
}

template <class T, int LPH>
__global__ __launch_bounds__(256) void cache4_read_kernel(Store4Args a)
{
    const int lane = threadIdx.x & (kWave - 1), lh = lane & (LPH - 1), d0 = 8 * lh;
    const int t = blockIdx.x * (kWave / LPH) + lane / LPH;
    const int h = blockIdx.y * 4 + threadIdx.x / kWave;
    if (h >= 2 * a.at.Hkv || t >= a.T || d0 >= a.D) return;
    const bool is_v = h >= a.at.Hkv;
    const int hk = is_v ? h - a.at.Hkv : h;
    const long long slot = store4_slot(a, t);
    uint32_t word = 0u, numbers = 0u;                                // a slot outside the cache: zeros
    if (slot >= 0) {
        const int r = static_cast<int>(slot) & ((1 << a.at.page_shift) - 1);
        const uint8_t* piece = a.cache + a.at.at(slot >> a.at.page_shift, hk);
        word = *reinterpret_cast<const uint32_t*>(piece + (is_v ? a.at.value_word(r, lh) : a.at.key_row(r) + 4 * lh));
        numbers = *reinterpret_cast<const uint32_t*>(piece + a.at.numbers(r) + (is_v ? 4 : 0));
    }
    const float s = T::widen(static_cast<uint16_t>(numbers & 0xFFFFu)), m = T::widen(static_cast<uint16_t>(numbers >> 16));
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(static_cast<float>(word >> (4 * (e >> 1) + 16 * (e & 1)) & 15u), s, m);
    uint16_t* out = (is_v ? a.v_out : a.k_out) + (static_cast<size_t>(t) * a.at.Hkv + hk) * a.D + d0;
    *reinterpret_cast<v4u*>(out) = narrow8<T>(x);
}

template <class T, int LPH>
int launch_store4(const Store4Args& a, bool write, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(divup(a.T, kWave / LPH)), static_cast<unsigned>(divup(2 * a.at.Hkv, 4)));
    if (write) cache4_write_kernel<T, LPH><<<grid, 64 * std::min(4, 2 * a.at.Hkv), 0, s>>>(a);
    else cache4_read_kernel<T, LPH><<<grid, 64 * std::min(4, 2 * a.at.Hkv), 0, s>>>(a);
    return launch_status();
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
    if (!cache4_shape_ok(Hkv, D, pages, page_size) || !k || !v || !cache || !slots || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(cache)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    for (long long st : {k_token, k_head, v_token, v_head})
        if (st < 0 || st % 8 != 0) return FORGE_EINVAL;
    const Store4Args a{k, v, nullptr, nullptr, cache, slots, k_token, k_head, v_token, v_head,
                       static_cast<long long>(pages) * page_size,
                       {cache4_units(D), __builtin_ctz(static_cast<unsigned>(page_size)), Hkv}, T, D};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_store4<Fp16>(a, true, s) : launch_store4<Bf16>(a, true, s);
}

extern "C" int forge_cache4_read(const uint8_t* cache, const int32_t* slots, uint16_t* k, uint16_t* v, int T, int Hkv, int D,
                                 int pages, int page_size, int dtype, void* stream)
{
    if (T <= 0 || Hkv <= 0 || D <= 0) return FORGE_OK;
    if (!cache4_shape_ok(Hkv, D, pages, page_size) || !k || !v || !cache || !slots || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(cache)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    const Store4Args a{nullptr, nullptr, k, v, const_cast<uint8_t*>(cache), slots, 0, 0, 0, 0,
                       static_cast<long long>(pages) * page_size,
                       {cache4_units(D), __builtin_ctz(static_cast<unsigned>(page_size)), Hkv}, T, D};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_store4<Fp16>(a, false, s) : launch_store4<Bf16>(a, false, s);
}
