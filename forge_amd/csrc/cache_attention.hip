// Attention of a few new tokens per sequence over a paged cache: one token (decode) or a tree of up to
// 64 drafted tokens, with grouped heads.
//
// Row t of sequence b sees the cache positions before cache_lens[b] and those drafted tokens j, which lie in
// the cache at cache_lens[b] + j, whose bit j is set in tree[b, t] (without a tree: j <= t). A row that
// sees nothing gives zeros.
//
// Bound: reading the cache. A KV head's rows (T tokens x Hq / Hkv heads) are taken together, up to 128 in a
// workgroup of RS x KS waves (32 rows each), so that K and V are read once for them; the keys are split
// over workgroups in chunks of equal length, whatever the sequence's, and a chunk's tiles, which come by
// LDS DMA into two buffers, over the KS waves of a row set. The waves' results are joined in LDS; the chunks'
// go as FP32 to the workspace and are joined by a second kernel, in a fixed order. 16 sequences with 16 drafts of
// 32 / 8 heads of 128 over 278 thousand keys: 252 us, 4.28 TB/s; one token over 1000 keys 9.4 (6.9 and 1.9 in two launches).
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

// Read in place of rows past the last key and on pages that the cache does not have.
__device__ const uint4 kZeroRow[32] = {};

__device__ __forceinline__ int cache_keys(const CacheArgs& a, int b) {
    const long long cap = static_cast<long long>(a.width) << a.page_shift;
    return static_cast<int>(min(static_cast<long long>(max(a.lens[b], 0)) + a.T, cap));
}

// LDS of the tiles, in which the waves' sums are left afterwards; the chunk's page numbers follow.
template <class T, int DP, int RS, int KS, int KB>
constexpr int kCacheLds = std::max<int>(4 * 32 * KS * KB * KvRows<DP>::kBytes,
                                        sizeof(typename AttnWave<T, DP, KB>::template Shared<RS * KS>));

template <class T, int DP, int RS, int KS, int KB>
__global__ __launch_bounds__(64 * RS * KS, DP > 128 ? 1 : 2) void cache_attention_kernel(CacheArgs a)
{
    using Rows = KvRows<DP>;
    constexpr int W = RS * KS, kKeys = 32 * KS * KB, kTile = kKeys * Rows::kBytes;
    constexpr int kIns = kKeys * Rows::kChunks / kWave / W;
    static_assert(kKeys * Rows::kChunks % (kWave * W) == 0, "a tile splits evenly over the waves");
    extern __shared__ __align__(1024) int8_t lds[];
    __shared__ int odd;
    int* page_of = reinterpret_cast<int*>(lds + kCacheLds<T, DP, RS, KS, KB>);

    const int group = a.group, rows = a.T * group;
    const int hk = blockIdx.x, chunk = blockIdx.y, b = udiv_magic(blockIdx.z, a.mg_sets), set = blockIdx.z - b * a.sets;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x & (kWave - 1);
    const int rs = wave / KS, ks = wave % KS;
    const int key0 = chunk * a.chunk, page_mask = (1 << a.page_shift) - 1, page0 = key0 >> a.page_shift;
    // the chunk's whole part of the table, so that its loads need not wait for the length
    const int last_page = min((key0 + a.chunk - 1) >> a.page_shift, a.width - 1);
    for (int p = page0 + threadIdx.x; p <= last_page; p += 64 * W) {
        const int pg = a.table[static_cast<size_t>(b) * a.width + p];
        page_of[p - page0] = pg >= 0 && pg < a.pages ? pg : -1;
    }

    const size_t token = static_cast<size_t>(a.Hkv) * a.D;
    // element offset of key j's row (of both tensors), or -1
    auto row_at = [&](int j) -> long long {
        const int pg = page_of[((key0 + j) >> a.page_shift) - page0];
        return pg < 0 ? -1LL
                      : static_cast<long long>((((static_cast<size_t>(pg) << a.page_shift) + ((key0 + j) & page_mask)) *
                                                token) + static_cast<size_t>(hk) * a.D);
    };
    auto row_of = [&](auto* base, int r) {                     // of q and out
        const int t = udiv_magic(r, a.mg_group);
        return base + ((static_cast<size_t>(b) * a.T + t) * a.Hq + hk * group + (r - t * group)) * a.D;
    };
    auto drafts_of = [&](int r) {                                    // the new tokens that row r sees
        const int t = udiv_magic(r, a.mg_group);
        return a.tree ? static_cast<unsigned long long>(a.tree[static_cast<size_t>(b) * a.T + t]) : ~0ull >> (63 - t);
    };

    AttnWave<T, DP, KB> w;
    if (threadIdx.x == 0) odd = -1;
    w.init();
    const int row = (set * RS + rs) * 32 + (lane & 31);
    const bool live = row < rows;
    w.load_q(row_of(a.q, row), live, a.D);
    const unsigned long long drafts = live ? drafts_of(row) : 0ull;
    const int keys = cache_keys(a, b), len = max(a.lens[b], 0), n = min(keys - key0, a.chunk);
    if (n <= 0) return;
    w.keys(keys);
    __syncthreads();
    const int open = len - key0;                                     // keys of this chunk that every row sees

    int dma_row[kIns];
    int ck[kIns], cv[kIns];
#pragma unroll
    for (int i = 0; i < kIns; i++) {
        const int c = (wave * kIns + i) * kWave + lane, p = c % Rows::kChunks;
        dma_row[i] = c / Rows::kChunks;
        ck[i] = 8 * (p ^ Rows::swz_k(dma_row[i]));
        cv[i] = 8 * (p ^ Rows::swz_v(dma_row[i]));
    }
    const uint32_t lds0 = lds_address(lds);
    auto load = [&](int t) {
        const uint32_t to = lds0 + (t & 1) * 2 * kTile + wave * kIns * 1024;
        const uint16_t* zero = reinterpret_cast<const uint16_t*>(kZeroRow);
#pragma unroll
        for (int i = 0; i < kIns; i++) {
            const int j = t * kKeys + dma_row[i];
            const long long at = j < n ? row_at(j) : -1LL;
            dma16_at(at >= 0 && ck[i] < a.D ? a.k + at + ck[i] : zero, to + i * 1024);
            dma16_at(at >= 0 && cv[i] < a.D ? a.v + at + cv[i] : zero, to + kTile + i * 1024);
        }
    };
    const float scale2 = a.scale * 1.44269504f;
    const int tiles = (n + kKeys - 1) / kKeys;
    const bool some = a.T > 1 || a.tree;                             // drafts that not every row sees
    load(0);
    for (int t = 0; t < tiles; t++) {
        wait_vm_lgkm<0>();
        lds_barrier();                                               // tile t is whole, tile t - 1 is read
        if (t + 1 < tiles) load(t + 1);
        const int k0 = t * kKeys + 32 * KB * ks;                     // this wave's keys of the tile
        const int8_t* at = lds + (t & 1) * 2 * kTile + 32 * KB * ks * Rows::kBytes;
        auto seen = [&](int kb) {
            const int d = open - (k0 + 32 * kb);                     // bits below d: the cache; from d on: drafts
            uint32_t bits = bits_to(d - 1);
            if (d < 32) bits |= d >= 0 ? static_cast<uint32_t>(drafts << d) : d > -64 ? static_cast<uint32_t>(drafts >> -d) : 0u;
            return bits & bits_to(n - 1 - (k0 + 32 * kb));
        };
        if (some && (t + 1) * kKeys > open)                          // (what lies past the last key is zeros)
            w.template take_odd_values<W, KS>(lds + (t & 1) * 2 * kTile + kTile, at + kTile, wave, t, &odd, seen);
        v16f s[KB];
        w.scores(at, s);
        w.finish(s, at + kTile, scale2, t == 0, k0 + 32 * KB > min(open, n), seen);
    }

    wait_vm_lgkm<0>();
    __syncthreads();
    auto* sh = reinterpret_cast<typename AttnWave<T, DP, KB>::template Shared<W>*>(lds);
    w.leave(sh, wave, live);
    __syncthreads();
    const bool whole = keys <= a.chunk;                              // the only chunk: the result itself
    const size_t part0 = ((static_cast<size_t>(b) * a.Hkv + hk) * a.chunks + chunk) * rows;
    if (!live) return;
    float* part = a.part + (part0 + row) * a.D;
    uint16_t* out = row_of(a.out, row);
    w.template join<KS>(sh, wave, [&](int j, int e, v4f s, float m, float l) {
        const int d = 32 * j + 8 * e + 4 * (lane >> 5);
        if (d >= a.D) return;
        if (whole) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            *reinterpret_cast<v2u*>(out + d) = v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
        } else {
            *reinterpret_cast<v4f*>(part + d) = s;
            if (d == 0) {
                a.stat[(part0 + row) * 2] = m;
                a.stat[(part0 + row) * 2 + 1] = l;
            }
        }
    });
}

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

inline int cache_row(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256; }

// Chunks such that sequences of the table's length make about a workgroup per CU, of as many keys as there are
// rows at least (a chunk's sums are as large as its keys and values then), in whole tiles of 128. us, with a
// third of that length / this: one token of 32 heads over 16000 27.8 / 21.0, 61 tokens of 32 heads over 16000 51 / 32.5;
// 4 trees of 61 over 3001, 17, 0 and 2048 with chunks of 128 19.7, of the 488 rows 15.
CachePlan cache_plan(int B, int T, int Hq, int Hkv, long long max_keys) {
    CachePlan p;
    const int rows = T * (Hq / Hkv);
    for (p.sets = 1; 32 * p.sets < rows && p.sets < 4;) p.sets *= 2;
    const long long heads = static_cast<long long>(B) * Hkv * divup(rows, 32 * p.sets);
    const long long want = std::max<long long>(1, divupll(default_cu_count(), heads));
    const long long chunk = divupll(std::max<long long>(divupll(max_keys, want), rows), 128) * 128;
    const long long most = std::max<long long>(kCacheMaxChunk, divupll(divupll(max_keys, kGridRows), 128) * 128);
    p.chunk = static_cast<int>(std::min(chunk, most));
    p.chunks = static_cast<int>(std::max<long long>(1, divupll(max_keys, p.chunk)));
    return p;
}

size_t cache_floats(int B, int T, int Hq, int D, const CachePlan& p) {
    return p.chunks == 1 ? 0 : static_cast<size_t>(B) * T * Hq * p.chunks * (D + 2);
}

template <class T, int DP, int RS, int KS, int KB>
int launch_cache(CacheArgs a, hipStream_t s) {
    constexpr int LPR = DP <= 64 ? 16 : DP <= 128 ? 32 : 64, kMost = kCacheLds<T, DP, RS, KS, KB> + 4 * (kCacheMaxChunk + 128 + 2);
    static_assert(kMost <= 159 * 1024, "tiles, sums and page numbers fit");
    static_assert(divupll(kCacheMaxKeys, kGridRows) <= kCacheMaxChunk + 128, "the longest table's chunks are a grid's rows");
    const int lds = kCacheLds<T, DP, RS, KS, KB> + 4 * ((a.chunk >> a.page_shift) + 2);
    const int rows = a.T * (a.Hq / a.Hkv);
    a.sets = divup(rows, 32 * RS);
    a.mg_sets = udiv_multiplier(a.sets);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&cache_attention_kernel<T, DP, RS, KS, KB>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (attr != hipSuccess) return static_cast<int>(attr);
    // as many sequences at a time as a grid has rows
    const long long total = a.B, most = kGridRows / a.sets;
    const size_t parts = static_cast<size_t>(a.T) * a.Hq * a.chunks;     // of a sequence
    for (long long b = 0; b < total; b += most) {
        a.B = static_cast<int>(std::min(most, total - b));
        const dim3 grid(static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.B * a.sets));
        cache_attention_kernel<T, DP, RS, KS, KB><<<grid, 64 * RS * KS, lds, s>>>(a);
        int st = launch_status();
        if (st == FORGE_OK && a.chunks > 1) {
            const dim3 rows_grid(static_cast<unsigned>(divup(a.Hq, 4)), static_cast<unsigned>(a.T), static_cast<unsigned>(a.B));
            cache_join_kernel<T, LPR><<<rows_grid, 256, 0, s>>>(a);
            st = launch_status();
        }
        if (st != FORGE_OK) return st;
        const size_t q = static_cast<size_t>(a.B) * a.T * a.Hq * a.D;
        a.q += q;
        a.out += q;
        a.table += static_cast<size_t>(a.B) * a.width;
        a.lens += a.B;
        if (a.tree) a.tree += static_cast<size_t>(a.B) * a.T;
        if (a.part) {
            a.part += a.B * parts * a.D;
            a.stat += a.B * parts * 2;
        }
    }
    return FORGE_OK;
}

// Waves by 32-row sets, then by keys, up to 8 (4 at 256 values a head, whose sums take 128 registers a lane);
// tiles of 64 or 128 keys, 128 KB of LDS at most for two of K and V.
template <class T>
int launch_cache(const CacheArgs& a, int sets, hipStream_t s) {
    switch (cache_row(a.D)) {
    case 64:
        if (sets == 1) return launch_cache<T, 64, 1, 4, 1>(a, s);
        return sets == 2 ? launch_cache<T, 64, 2, 4, 1>(a, s) : launch_cache<T, 64, 4, 2, 2>(a, s);
    case 96:
        if (sets == 1) return launch_cache<T, 96, 1, 4, 1>(a, s);
        return sets == 2 ? launch_cache<T, 96, 2, 4, 1>(a, s) : launch_cache<T, 96, 4, 2, 2>(a, s);
    case 128:
        if (sets == 1) return launch_cache<T, 128, 1, 4, 1>(a, s);
        return sets == 2 ? launch_cache<T, 128, 2, 4, 1>(a, s) : launch_cache<T, 128, 4, 2, 2>(a, s);
    default:
        if (sets == 1) return launch_cache<T, 256, 1, 2, 1>(a, s);
        return sets == 2 ? launch_cache<T, 256, 2, 2, 1>(a, s) : launch_cache<T, 256, 4, 1, 2>(a, s);
    }
}

// Rows (up to the last set's end) and heads are divided by the heads of a group in udiv_magic's range. The row sets of a
// sequence are then under 2^13, a few sequences' at least fit a grid, and their number too is divided in that range.
bool cache_shape_ok(int B, int T, int Hq, int Hkv, int D) {
    if (B <= 0 || T <= 0 || T > kCacheMaxTokens || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D % 8 != 0 || D > 256)
        return false;
    const long long group = Hq / Hkv;
    return static_cast<long long>(B) * T * Hq <= INT_MAX && (T * group + 128) * group < 1LL << 32 && (Hq + 4LL) * group < 1LL << 32;
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_cache_attention_workspace_size(int B, int T, int Hq, int Hkv, int D, long long max_keys) {
    if (!cache_shape_ok(B, T, Hq, Hkv, D) || max_keys <= 0 || max_keys > kCacheMaxKeys) return 0;
    return 4 * cache_floats(B, T, Hq, D, cache_plan(B, T, Hq, Hkv, max_keys));
}

extern "C" int forge_cache_attention(const uint16_t* q, const uint16_t* k_cache, const uint16_t* v_cache,
                                     const int32_t* page_table, const int32_t* cache_lens, const int64_t* tree,
                                     uint16_t* out, int B, int T, int Hq, int Hkv, int D, int pages, int page_size,
                                     int table_width, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                     void* stream)
{
    if (B <= 0 || T <= 0 || Hq <= 0 || D <= 0) return FORGE_OK;
    if (!cache_shape_ok(B, T, Hq, Hkv, D) || !q || !k_cache || !v_cache || !page_table || !cache_lens || !out ||
        pages <= 0 || page_size <= 0 || (page_size & (page_size - 1)) != 0 || table_width <= 0 ||
        !(scale > 0.0f && scale < INFINITY) || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k_cache), static_cast<const void*>(v_cache),
                          static_cast<const void*>(out), static_cast<const void*>(workspace)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    const long long max_keys = static_cast<long long>(table_width) * page_size;
    if (max_keys > kCacheMaxKeys) return FORGE_EINVAL;
    const CachePlan p = cache_plan(B, T, Hq, Hkv, max_keys);
    const size_t floats = cache_floats(B, T, Hq, D, p);
    if (floats && (!workspace || workspace_bytes < 4 * floats)) return FORGE_EINVAL;
    float* part = static_cast<float*>(workspace);
    const size_t parts = static_cast<size_t>(B) * T * Hq * p.chunks;
    const CacheArgs a{q, k_cache, v_cache, page_table, cache_lens, tree, out, part, part ? part + parts * D : nullptr,
                      B, T, Hq, Hkv, D, pages, __builtin_ctz(static_cast<unsigned>(page_size)), table_width,
                      p.chunk, p.chunks, Hq / Hkv, 1, udiv_multiplier(Hq / Hkv), 0u, scale};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_cache<Fp16>(a, p.sets, s) : launch_cache<Bf16>(a, p.sets, s);
}
