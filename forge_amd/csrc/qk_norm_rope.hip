// Norm of the query and key heads and rotation by their positions in one pass, with the write of
// keys and values into a paged cache.
//
// Per head of D values: y = x / sqrt(mean(x^2) + eps) * weight (a side without a weight is not
// normed), then for the pairs (a, b) of its first R values, (i, i + R/2) or neighbours (2i, 2i + 1),
// a' = a cos - b sin, b' = b cos + a sin with the table row of the token's position. FP32 inside,
// rounded once. Bound: memory; every value is read and written once, 16 bytes a lane: 16384 tokens of 64 + 8
// heads of 128 with their values into the cache 142 us, 680 MB at 4.8 TB/s, the rate of a copy; 8 tokens 3.3 us.
#include "float16_types.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

struct QkArgs {
    const uint16_t *q, *k, *v, *qw, *kw;
    const float *cos, *sin;
    const int32_t *pos, *slots;
    uint16_t *q_out, *k_out, *k_cache, *v_cache;
    long long q_token, q_head, k_token, k_head, v_token, v_head, cache_rows;
    int T, Hq, Hkv, D, half, table_rows, groups;   // half: R / 2; groups: waves' worth of heads per token
    float eps;
};

// A head is LPH lanes of 8 values. Pairs (i, i + R/2): the other half's values are loaded as well
// (they are in the cache line the neighbouring lanes load), which is cheaper than exchanging eight registers.
template <class T, int LPH, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs a)
{
    constexpr int kHeads = kWave / LPH;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int lh = lane & (LPH - 1), d0 = 8 * lh;
    const long long t = blockIdx.x;
    const bool in_d = d0 < a.D, rot = d0 < 2 * a.half;
    const int heads = a.Hq + a.Hkv + (a.v_cache ? a.Hkv : 0);

    // this lane's pair partner, and the cos and +-sin of its 8 values
    int partner = d0;
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) { c[e] = 1.0f; s[e] = 0.0f; }
    const int p = a.pos[t];
    const bool known = p >= 0 && p < a.table_rows;
    if (rot) {
        const size_t row = static_cast<size_t>(known ? p : 0) * a.half;
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float ce = a.cos[row + d0 / 2 + e], se = a.sin[row + d0 / 2 + e];
                c[2 * e] = c[2 * e + 1] = ce;
                s[2 * e] = -se;
                s[2 * e + 1] = se;
            }
        } else {
            const bool first = d0 < a.half;
            const int i0 = first ? d0 : d0 - a.half;
            partner = first ? d0 + a.half : i0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                c[e] = a.cos[row + i0 + e];
                const float se = a.sin[row + i0 + e];
                s[e] = first ? -se : se;
            }
        }
        // a position that the table does not have gives NaN, not another position's rotation
        if (!known) {
#pragma unroll
            for (int e = 0; e < 8; e++) c[e] = __uint_as_float(0x7FC00000u);
        }
    }
    long long slot = -1;
    if (a.slots) {
        slot = a.slots[t];
        if (slot >= a.cache_rows) slot = -1;
    }
    const v4u zero = {0u, 0u, 0u, 0u};
    for (int grp = blockIdx.y * 4 + wave; grp < a.groups; grp += 4 * gridDim.y) {
        const int h = grp * kHeads + lane / LPH;
        const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv, live = h < heads && in_d;
        const int hk = is_q ? 0 : h - a.Hq - (is_v ? a.Hkv : 0);
        const uint16_t* src = is_q ? a.q + t * a.q_token + h * a.q_head
                                   : is_v ? a.v + t * a.v_token + hk * a.v_head : a.k + t * a.k_token + hk * a.k_head;
        const uint16_t* wgt = is_q ? a.qw : a.kw;
        const v4u own = live ? *reinterpret_cast<const v4u*>(src + d0) : zero;
        v4u other = zero;
        if (!INTERLEAVED && live && rot) other = *reinterpret_cast<const v4u*>(src + partner);
        float x[8], o[8];
        widen8<T>(own, x);
        widen8<T>(other, o);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[e], x[e], ss);
#pragma unroll
        for (int d = 1; d < LPH; d <<= 1) ss += __shfl_xor(ss, d, kWave);
        // BF16 heads whose squares FP32 does not hold (values from about 2^60 on): once more in 64 bits
        float inv = 1.0f / sqrtf(ss / static_cast<float>(a.D) + a.eps);
        if (T::kWide && __any(ss == INFINITY)) {
            double sd = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) sd += static_cast<double>(x[e]) * x[e];
            for (int d = 1; d < LPH; d <<= 1) sd += __shfl_xor(sd, d, kWave);
            if (ss == INFINITY) inv = static_cast<float>(1.0 / sqrt(sd / a.D + a.eps));
        }
        if (!live) continue;
        if (is_v) {
            if (slot >= 0)
                *reinterpret_cast<v4u*>(a.v_cache + (static_cast<size_t>(slot) * a.Hkv + hk) * a.D + d0) = own;
            continue;
        }
        if (wgt) {
            float w[8];
            widen8<T>(*reinterpret_cast<const v4u*>(wgt + d0), w);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= inv * w[e];
            if (!INTERLEAVED && rot) {
                widen8<T>(*reinterpret_cast<const v4u*>(wgt + partner), w);
#pragma unroll
                for (int e = 0; e < 8; e++) o[e] *= inv * w[e];
            }
        }
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float b = INTERLEAVED ? x[e ^ 1] : o[e];
            y[e] = rot ? __builtin_fmaf(x[e], c[e], b * s[e]) : x[e];
        }
        const v4u r = narrow8<T>(y);
        if (is_q) {
            *reinterpret_cast<v4u*>(a.q_out + (t * a.Hq + h) * a.D + d0) = r;
        } else {
            if (a.k_out) *reinterpret_cast<v4u*>(a.k_out + (t * a.Hkv + hk) * a.D + d0) = r;
            if (slot >= 0) *reinterpret_cast<v4u*>(a.k_cache + (static_cast<size_t>(slot) * a.Hkv + hk) * a.D + d0) = r;
        }
    }
}

template <class T, int LPH>
int launch_qk(QkArgs a, bool interleaved, hipStream_t s) {
    a.groups = divup(a.Hq + a.Hkv + (a.v_cache ? a.Hkv : 0), kWave / LPH);
    // One head group per wave while tokens alone do not fill the card; the table row is loaded once
    // for more of them after that.
    const int split = a.T < 1024 ? divup(a.groups, 4) : 1;
    const dim3 grid(static_cast<unsigned>(a.T), static_cast<unsigned>(split));
    if (interleaved) qk_norm_rope_kernel<T, LPH, true><<<grid, 256, 0, s>>>(a);
    else qk_norm_rope_kernel<T, LPH, false><<<grid, 256, 0, s>>>(a);
    return launch_status();
}

template <class T>
int launch_qk(const QkArgs& a, bool interleaved, hipStream_t s) {
    if (a.D <= 64) return launch_qk<T, 8>(a, interleaved, s);
    if (a.D <= 128) return launch_qk<T, 16>(a, interleaved, s);
    return launch_qk<T, 32>(a, interleaved, s);
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" int forge_qk_norm_rope(const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* q_weight,
                                  const uint16_t* k_weight, const float* cos, const float* sin, const int32_t* positions,
                                  uint16_t* q_out, uint16_t* k_out, uint16_t* k_cache, uint16_t* v_cache,
                                  const int32_t* slots, long long cache_rows, int T, int Hq, int Hkv, int D, int R,
                                  int table_rows, long long q_token, long long q_head, long long k_token,
                                  long long k_head, long long v_token, long long v_head, float eps, int interleaved,
                                  int dtype, void* stream)
{
    if (T <= 0 || D <= 0 || Hq < 0 || Hkv < 0 || Hq + Hkv == 0) return FORGE_OK;
    const bool cache = k_cache || v_cache;
    if (T > grid_limit(256) || D % 8 != 0 || D > 256 || R < 0 || R > D || R % 16 != 0 || Hq > 65535 || Hkv > 65535 || !positions ||
        (R > 0 && (!cos || !sin || table_rows <= 0)) || (Hq > 0 && (!q || !q_out)) || (Hkv > 0 && !k) ||
        (Hkv > 0 && !k_out && !cache) || (cache && (!k_cache || !v_cache || !v || !slots || cache_rows < 0)) ||
        (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k), static_cast<const void*>(v),
                          static_cast<const void*>(q_weight), static_cast<const void*>(k_weight),
                          static_cast<const void*>(q_out), static_cast<const void*>(k_out),
                          static_cast<const void*>(k_cache), static_cast<const void*>(v_cache)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    for (long long st : {q_token, q_head, k_token, k_head, v_token, v_head})
        if (st < 0 || st % 8 != 0) return FORGE_EINVAL;
    const QkArgs a{q, k, v, q_weight, k_weight, cos, sin, positions, cache ? slots : nullptr,
                   q_out, k_out, k_cache, v_cache, q_token, q_head, k_token, k_head, v_token, v_head, cache_rows,
                   T, Hq, Hkv, D, R / 2, table_rows, 0, eps};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_qk<Fp16>(a, interleaved != 0, s) : launch_qk<Bf16>(a, interleaved != 0, s);
}
