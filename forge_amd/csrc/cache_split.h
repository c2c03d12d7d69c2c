// What the attention kernels over a paged cache share: their arguments, the split of the keys into chunks and the join
// of the chunks' results.
#pragma once

#include "attn_tile.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr int kCacheMaxChunk = 2048;   // keys; a chunk's pages are looked up in LDS (128 more for the longest tables)
constexpr int kCacheMaxTokens = 64;
constexpr long long kCacheMaxKeys = 1LL << 27;
constexpr int kGridRows = 65535;       // of a grid's second and third dimension

struct CachePlan {
    int chunk, chunks;   // keys of a chunk; chunks of the longest sequence
    int sets;            // 32-row sets of a workgroup: 1, 2 or 4
};

struct CacheArgs {
    const uint16_t *q, *k, *v;
    const int32_t *table, *lens;
    const int64_t* tree;
    uint16_t* out;
    float *part, *stat;  // (B, Hkv, chunks, rows, D) sums and (.., rows, 2) maxima and sums of the chunks
    int B, T, Hq, Hkv, D, pages, page_shift, width, chunk, chunks, group, sets;
    uint32_t mg_group, mg_sets;   // udiv_magic multipliers
    float scale;
};

__device__ __forceinline__ int cache_keys(const CacheArgs& a, int b) {
    const long long cap = static_cast<long long>(a.width) << a.page_shift;
    return static_cast<int>(min(static_cast<long long>(max(a.lens[b], 0)) + a.T, cap));
}

namespace {   // a kernel of each source's own

// A wave joins one row's chunks: LPR lanes of 4 values take every (64 / LPR)-th chunk, four in flight, with the
// running maximum of a softmax, and the lanes' sums are joined in a fixed order. The first ones are loaded before the
// sequence's length is there.
template <class T, int LPR>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheArgs a)
{
    constexpr int kSets = kWave / LPR;
    const int lane = threadIdx.x & (kWave - 1), sub = lane / LPR, d = 4 * (lane % LPR);
    const int t = blockIdx.y, b = blockIdx.z, h = blockIdx.x * 4 + threadIdx.x / kWave;
    if (h >= a.Hq) return;
    const int rows = a.T * a.group;
    const int hk = udiv_magic(h, a.mg_group), r = t * a.group + h - hk * a.group;
    const size_t first = (static_cast<size_t>(b) * a.Hkv + hk) * a.chunks;
    const bool in = d < a.D;
    float m = kNoScore, l = 0.0f;
    v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
    int used = a.chunks;
    for (int c0 = sub; c0 - sub < used; c0 += 4 * kSets) {
        v4f x[4];
        v2f st[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const size_t at = (first + min(c0 + u * kSets, a.chunks - 1)) * rows + r;
            st[u] = *reinterpret_cast<const v2f*>(a.stat + at * 2);
            x[u] = *reinterpret_cast<const v4f*>(a.part + at * a.D + (in ? d : 0));
        }
        if (c0 == sub) {
            used = (cache_keys(a, b) + a.chunk - 1) / a.chunk;
            if (used <= 1) return;                                   // the only chunk has written the result
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (c0 + u * kSets >= used) continue;
            const float mn = fmaxf(m, st[u][0]);
            const float f = __builtin_amdgcn_exp2f(m - mn), g = __builtin_amdgcn_exp2f(st[u][0] - mn);
            m = mn;
            l = __builtin_fmaf(l, f, st[u][1] * g);
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = __builtin_fmaf(s[e], f, x[u][e] * g);
        }
    }
#pragma unroll
    for (int o = LPR; o < kWave; o <<= 1) {
        const float om = __shfl_xor(m, o, kWave), mn = fmaxf(m, om);
        const float f = __builtin_amdgcn_exp2f(m - mn), g = __builtin_amdgcn_exp2f(om - mn);
        m = mn;
        l = l * f + __shfl_xor(l, o, kWave) * g;
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] = s[e] * f + __shfl_xor(s[e], o, kWave) * g;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    if (in && sub == 0)
        *reinterpret_cast<v2u*>(a.out + ((static_cast<size_t>(b) * a.T + t) * a.Hq + h) * a.D + d) =
            v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
}

}  // namespace

inline size_t cache_floats(int B, int T, int Hq, int D, const CachePlan& p) {
    return p.chunks == 1 ? 0 : static_cast<size_t>(B) * T * Hq * p.chunks * (D + 2);
}

// Rows (up to the last set's end) and heads are divided by the heads of a group in udiv_magic's range. The row sets of a
// sequence are then under 2^13, a few sequences' at least fit a grid, and their number too is divided in that range.
inline bool cache_shape_ok(int B, int T, int Hq, int Hkv, int D) {
    if (B <= 0 || T <= 0 || T > kCacheMaxTokens || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D % 8 != 0 || D > 256)
        return false;
    const long long group = Hq / Hkv;
    return static_cast<long long>(B) * T * Hq <= INT_MAX && (T * group + 128) * group < 1LL << 32 && (Hq + 4LL) * group < 1LL << 32;
}

}  // namespace forge_amd
