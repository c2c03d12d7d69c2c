// What the attention kernels over a paged cache share: their arguments and limits.
#pragma once

#include "attn_tile.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr int kCacheMaxChunk = 2048;   // keys; a chunk's pages are looked up in LDS (128 more for the longest tables)
constexpr int kCacheMaxTokens = 64;
constexpr long long kCacheMaxKeys = 1LL << 27;
constexpr int kGridRows = 65535;       // of a grid's second and third dimension

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

// Rows (up to the last set's end) and heads are divided by the heads of a group in udiv_magic's range. The row sets of a
// sequence are then under 2^13, a few sequences' at least fit a grid, and their number too is divided in that range.
inline bool cache_shape_ok(int B, int T, int Hq, int Hkv, int D) {
    if (B <= 0 || T <= 0 || T > kCacheMaxTokens || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D % 8 != 0 || D > 256)
        return false;
    const long long group = Hq / Hkv;
    return static_cast<long long>(B) * T * Hq <= INT_MAX && (T * group + 128) * group < 1LL << 32 && (Hq + 4LL) * group < 1LL << 32;
}

}  // namespace forge_amd
