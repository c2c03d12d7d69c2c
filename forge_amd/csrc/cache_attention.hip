// Attention of a few new tokens per sequence over a paged cache: one token (decode) or a tree of up to
// 64 drafted tokens, with grouped heads.
//
// Row t of sequence b sees the cache positions before cache_lens[b] and those drafted tokens j, which lie in
// the cache at cache_lens[b] + j, whose bit j is set in tree[b, t] (without a tree: j <= t). A row that
// sees nothing gives zeros.
//
// Bound: reading the cache. A KV head's rows (T tokens x Hq / Hkv heads) are taken together, 32 or 64
// to a wave, so that K and V are read once for them; the keys are split over workgroups in chunks
// of equal length, whatever the sequence's, and in a chunk over the waves, each with tiles of 32
// keys in two LDS buffers of its own (no barrier while it streams). The waves' results are joined in
// LDS; the chunks' go as FP32 to the workspace and are joined by a second kernel, in chunk order.
#include "attn_tile.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr int kCacheMaxChunk = 2048;   // keys; a chunk's pages are looked up in LDS
constexpr int kCacheMaxTokens = 64;

struct CachePlan {
    int chunk, chunks;   // keys of a chunk; chunks of the longest sequence
    int sets;            // 32-row sets per wave
};

struct CacheArgs {
    const uint16_t *q, *k, *v;
    const int32_t *table, *lens;
    const int64_t* tree;
    uint16_t* out;
    float *part, *stat;  // (B, Hkv, chunks, rows, D) sums and (.., rows, 2) maxima and sums of the chunks
    int B, T, Hq, Hkv, D, pages, page_shift, width, chunk, chunks;
    float scale;
};

// Read in place of rows past the last key and on pages that the cache does not have.
__device__ const uint4 kZeroRow[32] = {};

__device__ __forceinline__ int cache_keys(const CacheArgs& a, int b) {
    const long long cap = static_cast<long long>(a.width) << a.page_shift;
    return static_cast<int>(min(static_cast<long long>(max(a.lens[b], 0)) + a.T, cap));
}

template <class T, int DP, int RB, int W>
__global__ __launch_bounds__(64 * W) void cache_attention_kernel(CacheArgs a)
{
    using Rows = KvRows<DP>;
    constexpr int kKeys = 32, kTile = kKeys * Rows::kBytes, kIns = kKeys * Rows::kChunks / kWave;
    constexpr int kWaveLds = 4 * kTile, kPitch = DP + 4;
    static_assert(32 * RB * kPitch * 4 <= kWaveLds + 32 * RB * 16, "the waves' sums fit the tiles' LDS and its pad");
    extern __shared__ __align__(1024) int8_t lds[];
    __shared__ int page_of[kCacheMaxChunk + 2];
    __shared__ float stat_m[W][32 * RB], stat_l[W][32 * RB];
    __shared__ int odd_rows;

    const int group = a.Hq / a.Hkv, rows = a.T * group, sets = (rows + 32 * RB - 1) / (32 * RB);
    int id = blockIdx.x;
    const int hk = id % a.Hkv; id /= a.Hkv;
    const int set = id % sets; id /= sets;
    const int chunk = id % a.chunks, b = id / a.chunks;
    const int keys = cache_keys(a, b), len = max(a.lens[b], 0);
    const int key0 = chunk * a.chunk, n = min(keys - key0, a.chunk);
    if (n <= 0) return;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x & (kWave - 1);
    const int page_mask = (1 << a.page_shift) - 1, page0 = key0 >> a.page_shift;
    const int last_page = (key0 + n - 1) >> a.page_shift;
    for (int p = page0 + threadIdx.x; p <= last_page; p += 64 * W) {
        const int pg = a.table[static_cast<size_t>(b) * a.width + p];
        page_of[p - page0] = pg >= 0 && pg < a.pages ? pg : -1;
    }
    if (threadIdx.x == 0) odd_rows = 0;
    __syncthreads();

    const size_t token = static_cast<size_t>(a.Hkv) * a.D;
    // element offset of key j's row (of both tensors), or -1
    auto row_at = [&](int j) -> long long {
        const int pg = page_of[((key0 + j) >> a.page_shift) - page0];
        return pg < 0 ? -1LL
                      : static_cast<long long>((((static_cast<size_t>(pg) << a.page_shift) + ((key0 + j) & page_mask)) *
                                                token) + static_cast<size_t>(hk) * a.D);
    };

    AttnWave<T, DP, RB, 1> w;
    w.init();
    unsigned long long bits[RB];
#pragma unroll
    for (int s = 0; s < RB; s++) {
        const int r = (set * RB + s) * 32 + (lane & 31), t = r / group, g = r - t * group;
        const bool live = r < rows;
        w.load_q(s, a.q + ((static_cast<size_t>(b) * a.T + t) * a.Hq + hk * group + g) * a.D, live, a.D);
        bits[s] = !live ? 0ull
                        : a.tree ? static_cast<unsigned long long>(a.tree[static_cast<size_t>(b) * a.T + t])
                                 : ~0ull >> (63 - t);
    }
    const int open = len - key0;                                     // keys of this chunk that every row sees
    auto sees = [&](int s, int j) {
        const int d = j - open;
        return j < n && (d < 0 || (bits[s] >> (d & 63)) & 1ull);
    };

    int8_t* mine = lds + wave * kWaveLds;
    auto load = [&](int t, int buf) {
#pragma unroll
        for (int i = 0; i < kIns; i++) {
            const int c = i * kWave + lane, r = c / Rows::kChunks, p = c % Rows::kChunks;
            const int j = t * kKeys + r;
            const long long at = j < n ? row_at(j) : -1LL;
            const int ck = p ^ Rows::swz_k(r), cv = p ^ Rows::swz_v(r);
            const int8_t* zero = reinterpret_cast<const int8_t*>(kZeroRow);
            const int8_t* ks = at >= 0 && 8 * ck < a.D ? reinterpret_cast<const int8_t*>(a.k + at + 8 * ck) : zero;
            const int8_t* vs = at >= 0 && 8 * cv < a.D ? reinterpret_cast<const int8_t*>(a.v + at + 8 * cv) : zero;
            dma16(ks, mine + buf * 2 * kTile + i * 1024);
            dma16(vs, mine + buf * 2 * kTile + kTile + i * 1024);
        }
    };
    const float scale2 = a.scale * 1.44269504f;
    const int tiles = (n + kKeys - 1) / kKeys;
    if (wave < tiles) load(wave, 0);
    int buf = 0;
    for (int t = wave; t < tiles; t += W, buf ^= 1) {
        // the reads of the buffer that the next tile goes to are complete
        wait_lgkm0();
        compiler_fence();
        if (t + W < tiles) {
            load(t + W, buf ^ 1);
            wait_vmcnt<2 * kIns>();
        } else {
            wait_vmcnt<0>();
        }
        compiler_fence();
        const int8_t* ks = mine + buf * 2 * kTile;
        const int k0 = t * kKeys;
        if (k0 + kKeys > open || k0 + kKeys > n)
            w.template step<true>(ks, ks + kTile, scale2, [&](int s, int j) { return sees(s, k0 + j); });
        else
            w.template step<false>(ks, ks + kTile, scale2, [](int, int) { return true; });
    }

    // ---- join the waves, in wave order
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int s = 0; s < RB; s++) {
        const int r = 32 * s + (lane & 31);
        if (w.odd(s, (set * RB + s) * 32 + (lane & 31) < rows) && lane == 0) atomicOr(&odd_rows, 1);
        const float l = half_sum(w.l[s]);
        if (lane < 32) {
            stat_m[wave][r] = w.m[s];
            stat_l[wave][r] = l;
        }
#pragma unroll
        for (int j = 0; j < DP / 32; j++)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<v4f*>(sums + (wave * 32 * RB + r) * kPitch + 32 * j + 2 * e + 4 * (lane >> 5)) =
                    v4f{w.o[s][j][e], w.o[s][j][e + 1], w.o[s][j][e + 2], w.o[s][j][e + 3]};
    }
    __syncthreads();
    const bool whole = keys <= a.chunk;                              // the only chunk: the result itself
    const size_t part0 = (static_cast<size_t>(b) * a.Hkv + hk) * a.chunks + chunk;
    auto out_row = [&](int r) {
        const int t = r / group;
        return a.out + ((static_cast<size_t>(b) * a.T + t) * a.Hq + hk * group + (r - t * group)) * a.D;
    };
    if (odd_rows) {
        // some row's sum is not finite: every row again, key by key
        for (int i = wave; i < 32 * RB; i += W) {
            const int r = set * RB * 32 + i;
            if (r >= rows) break;
            const int t = r / group;
            const unsigned long long rb = a.tree ? static_cast<unsigned long long>(a.tree[static_cast<size_t>(b) * a.T + t])
                                                 : ~0ull >> (63 - t);
            float m, l, acc[(DP + 63) / 64];
            auto at = [&](const uint16_t* base, int j) {
                const long long o = row_at(j);
                return o < 0 ? reinterpret_cast<const uint16_t*>(kZeroRow) : base + o;
            };
            attn_row<T, DP>(
                a.q + ((static_cast<size_t>(b) * a.T + t) * a.Hq + hk * group + (r - t * group)) * a.D, a.D, n, scale2,
                [&](int j) { return at(a.k, j); }, [&](int j) { return at(a.v, j); },
                [&](int j) {
                    const int d = j - open;
                    return d < 0 || ((rb >> (d & 63)) & 1ull);
                },
                m, l, acc);
            for (int c = 0; c < (DP + 63) / 64; c++) {
                const int d = lane + 64 * c;
                if (d >= a.D) break;
                if (whole) out_row(r)[d] = narrow<T>(acc[c] * (l != 0.0f ? 1.0f / l : 0.0f));
                else a.part[(part0 * rows + r) * a.D + d] = acc[c];
            }
            if (!whole && lane == 0) {
                a.stat[(part0 * rows + r) * 2] = m;
                a.stat[(part0 * rows + r) * 2 + 1] = l;
            }
        }
        return;
    }
    const int quads = a.D / 4;
    for (int i = threadIdx.x; i < 32 * RB * quads; i += 64 * W) {
        const int lr = i / quads, d = 4 * (i - lr * quads), r = set * RB * 32 + lr;
        if (r >= rows) break;
        float m = kNoScore, l = 0.0f;
#pragma unroll
        for (int v = 0; v < W; v++) m = fmaxf(m, stat_m[v][lr]);
        v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < W; v++) {
            const float f = __builtin_amdgcn_exp2f(stat_m[v][lr] - m);
            l = __builtin_fmaf(f, stat_l[v][lr], l);
            const v4f x = *reinterpret_cast<const v4f*>(sums + (v * 32 * RB + lr) * kPitch + d);
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = __builtin_fmaf(f, x[e], s[e]);
        }
        if (whole) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            *reinterpret_cast<v2u*>(out_row(r) + d) = v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
        } else {
            *reinterpret_cast<v4f*>(a.part + (part0 * rows + r) * a.D + d) = s;
            if (d == 0) {
                a.stat[(part0 * rows + r) * 2] = m;
                a.stat[(part0 * rows + r) * 2 + 1] = l;
            }
        }
    }
}

// A wave joins one row's chunks.
template <class T>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheArgs a)
{
    const int lane = threadIdx.x & (kWave - 1);
    const long long id = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / kWave;
    const int group = a.Hq / a.Hkv, rows = a.T * group;
    if (id >= static_cast<long long>(a.B) * a.T * a.Hq) return;
    const int h = static_cast<int>(id % a.Hq), t = static_cast<int>(id / a.Hq % a.T);
    const int b = static_cast<int>(id / (static_cast<long long>(a.Hq) * a.T));
    const int keys = cache_keys(a, b);
    if (keys <= a.chunk && keys > 0) return;
    const int used = (keys + a.chunk - 1) / a.chunk, hk = h / group, r = t * group + h - hk * group;
    const size_t first = (static_cast<size_t>(b) * a.Hkv + hk) * a.chunks;
    float m = kNoScore;
    for (int c = 0; c < used; c++) m = fmaxf(m, a.stat[((first + c) * rows + r) * 2]);
    float l = 0.0f, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool in = 4 * lane < a.D;
    for (int c = 0; c < used; c++) {
        const size_t at = (first + c) * rows + r;
        const float f = __builtin_amdgcn_exp2f(a.stat[at * 2] - m);
        l = __builtin_fmaf(f, a.stat[at * 2 + 1], l);
        if (!in) continue;
        const v4f x = *reinterpret_cast<const v4f*>(a.part + at * a.D + 4 * lane);
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] = __builtin_fmaf(f, x[e], s[e]);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    if (in)
        *reinterpret_cast<v2u*>(a.out + id * a.D + 4 * lane) =
            v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
}

// Chunks such that the longest sequences make about three workgroups per CU, of 128 keys (one tile for
// each of four waves) at least.
CachePlan cache_plan(int B, int T, int Hq, int Hkv, long long max_keys) {
    CachePlan p;
    const int rows = T * (Hq / Hkv);
    p.sets = rows > 32 ? 2 : 1;
    const long long heads = static_cast<long long>(B) * Hkv * divup(rows, 32 * p.sets);
    const long long want = std::max<long long>(1, divupll(768, heads));
    const long long chunk = divupll(divupll(max_keys, want), 128) * 128;
    p.chunk = static_cast<int>(std::min<long long>(std::max<long long>(chunk, 128), kCacheMaxChunk));
    p.chunks = static_cast<int>(std::max<long long>(1, divupll(max_keys, p.chunk)));
    return p;
}

size_t cache_floats(int B, int T, int Hq, int D, const CachePlan& p) {
    return p.chunks == 1 ? 0 : static_cast<size_t>(B) * T * Hq * p.chunks * (D + 2);
}

template <class T, int DP, int RB, int W>
int launch_cache(const CacheArgs& a, hipStream_t s) {
    constexpr int kLds = W * (4 * 32 * KvRows<DP>::kBytes + 32 * RB * 16);
    const int rows = a.T * (a.Hq / a.Hkv);
    const long long wgs = static_cast<long long>(a.B) * a.Hkv * divup(rows, 32 * RB) * a.chunks;
    if (wgs > INT_MAX) return FORGE_EINVAL;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&cache_attention_kernel<T, DP, RB, W>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return static_cast<int>(attr);
    cache_attention_kernel<T, DP, RB, W><<<static_cast<unsigned>(wgs), 64 * W, kLds, s>>>(a);
    int st = launch_status();
    if (st != FORGE_OK || a.chunks == 1) return st;
    const long long all = static_cast<long long>(a.B) * a.T * a.Hq;
    cache_join_kernel<T><<<static_cast<unsigned>(divupll(all, 4)), 256, 0, s>>>(a);
    return launch_status();
}

template <class T, int RB>
int launch_cache(const CacheArgs& a, hipStream_t s) {
    if (a.D <= 64) return launch_cache<T, 64, RB, 4>(a, s);
    if (a.D <= 96) return launch_cache<T, 96, RB, 4>(a, s);
    if (a.D <= 128) return launch_cache<T, 128, RB, 4>(a, s);
    return launch_cache<T, 256, RB, 2>(a, s);
}

bool cache_shape_ok(int B, int T, int Hq, int Hkv, int D) {
    return B > 0 && T > 0 && T <= kCacheMaxTokens && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && D > 0 && D % 8 == 0 &&
           D <= 256 && static_cast<long long>(B) * T * Hq <= INT_MAX;
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_cache_attention_workspace_size(int B, int T, int Hq, int Hkv, int D, long long max_keys) {
    if (!cache_shape_ok(B, T, Hq, Hkv, D) || max_keys <= 0) return 0;
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
    if (max_keys > INT_MAX - kCacheMaxChunk) return FORGE_EINVAL;
    const CachePlan p = cache_plan(B, T, Hq, Hkv, max_keys);
    const size_t floats = cache_floats(B, T, Hq, D, p);
    if (floats && (!workspace || workspace_bytes < 4 * floats)) return FORGE_EINVAL;
    float* part = static_cast<float*>(workspace);
    const size_t parts = static_cast<size_t>(B) * T * Hq * p.chunks;
    const CacheArgs a{q, k_cache, v_cache, page_table, cache_lens, tree, out, part, part ? part + parts * D : nullptr,
                      B, T, Hq, Hkv, D, pages, __builtin_ctz(static_cast<unsigned>(page_size)), table_width,
                      p.chunk, p.chunks, scale};
    hipStream_t s = as_stream(stream);
    if (dtype == FORGE_FP16) return p.sets == 1 ? launch_cache<Fp16, 1>(a, s) : launch_cache<Fp16, 2>(a, s);
    return p.sets == 1 ? launch_cache<Bf16, 1>(a, s) : launch_cache<Bf16, 2>(a, s);
}
