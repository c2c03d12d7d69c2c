// The pages of a paged cache whose rows go on from one another, as a beam search's do after a selection.
//
// fork_pages: new row r goes on from row p of its group, parents[r] of it (none: the row ends). It names p's full pages again, without a copy;
// refs counts the names of each page. The page of its next token is p's own where p's first child takes it and nobody else
// names it, else the lowest free page not yet taken, the next for each row in order; the filled part of p's page is then to be copied (src, dst). Pages that
// this call frees are not taken by it, so no copied page is written. Counts are added to with integer atomics,
// whose order does not matter; everything else is in the rows' order.
//
// Bound: latency at few rows; two launches. First, a workgroup looks at the rows (first children, places among the takers) while others
// copy the counts and count free pages, a thousand each; then a workgroup per row finds its page and writes its table. copy_pages: memory.
#include "common.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr int kForkRows = 8192;      // rows that one workgroup looks at (first children in LDS)
constexpr int kForkThreads = 256;
constexpr int kForkPart = 1024;      // pages whose free ones are counted together

struct ForkArgs {
    const int32_t *table, *lens, *parents, *refs;
    int32_t *table_out, *lens_out, *refs_out, *slots, *src, *dst;
    int32_t *rank, *free;   // a row's place among those that take a page, or -1; free pages of a part
    int rows, group, width, pages, page_shift;
};

// Sum over the threads before this one, and over all (in *all), of a workgroup of 256.
__device__ __forceinline__ int sum_before(int x, int* all, int (&part)[4]) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int s = x;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(s, o, kWave);
        if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == kWave - 1) part[wave] = s;
    __syncthreads();
    int before = s - x;
#pragma unroll
    for (int w = 0; w < 4; w++) before += w < wave ? part[w] : 0;
    *all = part[0] + part[1] + part[2] + part[3];
    return before;
}

__device__ __forceinline__ int fork_parent(const ForkArgs& a, int r) {
    const int p = a.parents[r];
    return p >= 0 && p < a.group ? r - r % a.group + p : -1;
}
__device__ __forceinline__ int fork_len(const ForkArgs& a, int p) {
    const long long cap = static_cast<long long>(a.width) << a.page_shift;
    return p < 0 ? 0 : static_cast<int>(min(static_cast<long long>(max(a.lens[p], 0)), cap));
}
// The parent's page of the next token, or -1.
__device__ __forceinline__ int fork_last(const ForkArgs& a, int p, int at) {
    const int pg = at < a.width ? a.table[static_cast<size_t>(p) * a.width + at] : -1;
    return pg >= 0 && pg < a.pages ? pg : -1;
}

__global__ __launch_bounds__(kForkThreads) void fork_rows_kernel(ForkArgs a)
{
    __shared__ int part[4];
    if (blockIdx.x > 0) {                                            // a part of the counts
        const int at = (blockIdx.x - 1) * kForkPart + threadIdx.x;
        int n = 0, all;
#pragma unroll
        for (int i = 0; i < kForkPart / kForkThreads; i++) {
            const int pg = at + i * kForkThreads;
            if (pg >= a.pages) continue;
            const int x = a.refs[pg];
            a.refs_out[pg] = x;
            n += x == 0;
        }
        sum_before(n, &all, part);
        if (threadIdx.x == 0) a.free[blockIdx.x - 1] = all;
        return;
    }
    extern __shared__ int first[];                                   // a row's first child
    for (int r = threadIdx.x; r < a.rows; r += kForkThreads) first[r] = a.rows;
    __syncthreads();
    for (int r = threadIdx.x; r < a.rows; r += kForkThreads) {
        const int p = fork_parent(a, r);
        if (p >= 0) atomicMin(&first[p], r);
    }
    __syncthreads();
    int base = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kForkThreads) {
        const int r = r0 + threadIdx.x;
        bool take = false;
        if (r < a.rows) {
            const int p = fork_parent(a, r), at = fork_len(a, p) >> a.page_shift;
            if (p >= 0 && at < a.width) {
                const int last = fork_last(a, p, at);
                take = !(last >= 0 && first[p] == r && a.refs[last] == 1);
            }
        }
        int all;
        const int before = sum_before(take ? 1 : 0, &all, part);
        if (r < a.rows) a.rank[r] = take ? base + before : -1;
        base += all;
    }
}

__global__ __launch_bounds__(kForkThreads) void fork_table_kernel(ForkArgs a)
{
    __shared__ int part[4], mine;
    const int r = blockIdx.x, tid = threadIdx.x;
    const int p = fork_parent(a, r), len = fork_len(a, p), at = len >> a.page_shift;
    const int rank = a.rank[r];
    const bool room = p >= 0 && at < a.width;
    const int last = room ? fork_last(a, p, at) : -1;
    if (tid == 0) mine = rank < 0 ? last : -1;
    __syncthreads();
    if (rank >= 0) {
        // the part of the counts, then the page in it, that has the rank-th free one
        const int parts = (a.pages + kForkPart - 1) / kForkPart;
        int left = rank, which = -1;
        for (int i0 = 0; i0 < parts && which < 0; i0 += kForkThreads) {
            const int i = i0 + tid, x = i < parts ? a.free[i] : 0;
            int all;
            const int before = sum_before(x, &all, part);
            if (left < all) {
                __shared__ int found[2];
                if (before <= left && left < before + x) {
                    found[0] = i;
                    found[1] = left - before;
                }
                __syncthreads();
                which = found[0];
                left = found[1];
            } else {
                left -= all;
            }
        }
        if (which >= 0) {
            constexpr int kPer = kForkPart / kForkThreads;
            int n = 0, all;
            bool is[kPer];
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int pg = which * kForkPart + tid * kPer + i;
                is[i] = pg < a.pages && a.refs[pg] == 0;
                n += is[i];
            }
            int before = sum_before(n, &all, part);
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                if (is[i] && before == left) mine = which * kForkPart + tid * kPer + i;
                before += is[i];
            }
        }
        __syncthreads();
    }
    const int page = mine, in_page = len & ((1 << a.page_shift) - 1);
    if (tid == 0) {
        const bool copied = rank >= 0 && page >= 0 && last >= 0 && in_page > 0;
        a.lens_out[r] = len;
        a.slots[r] = page >= 0 ? (page << a.page_shift) + in_page : -1;
        a.src[r] = copied ? last : -1;
        a.dst[r] = copied ? page : -1;
    }
    // the old row's names go, the new row's come
    for (int i = tid; i < a.width; i += kForkThreads) {
        const int old = a.table[static_cast<size_t>(r) * a.width + i];
        int pg = p >= 0 && i < at ? a.table[static_cast<size_t>(p) * a.width + i] : room && i == at ? page : -1;
        if (pg < 0 || pg >= a.pages) pg = -1;
        a.table_out[static_cast<size_t>(r) * a.width + i] = pg;
        if (old != pg) {
            if (old >= 0 && old < a.pages) atomicAdd(&a.refs_out[old], -1);
            if (pg >= 0) atomicAdd(&a.refs_out[pg], 1);
        }
    }
}

// Whether two arrays of int32 share memory.
inline bool overlap(const int32_t* a, size_t na, const int32_t* b, size_t nb) { return a < b + nb && b < a + na; }

constexpr int kCopyTensors = 64;     // of a launch, by value
struct CopyArgs {
    uint8_t* tensor[kCopyTensors];
    const int32_t *src, *dst;
    long long page_bytes;
    int pairs, pages;
};

// A workgroup copies 4 KB of one page: blockIdx.x the piece, y the pair, z the tensor.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a)
{
    for (int i = blockIdx.y; i < a.pairs; i += gridDim.y) {
        const int s = a.src[i], d = a.dst[i];
        if (s < 0 || d < 0 || s >= a.pages || d >= a.pages || s == d) continue;
        const long long at = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 16;
        if (at >= a.page_bytes) continue;
        uint8_t* t = a.tensor[blockIdx.z];
        *reinterpret_cast<uint4*>(t + d * a.page_bytes + at) = *reinterpret_cast<const uint4*>(t + s * a.page_bytes + at);
    }
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_fork_pages_workspace_size(int rows, int pages) {
    if (rows <= 0 || rows > kForkRows || pages <= 0) return 0;
    return 4 * (static_cast<size_t>(rows) + divup(pages, kForkPart));
}

extern "C" int forge_fork_pages(const int32_t* page_table, const int32_t* cache_lens, const int32_t* parents, const int32_t* refs,
                                int32_t* table_out, int32_t* lens_out, int32_t* refs_out, int32_t* slots, int32_t* src,
                                int32_t* dst, int rows, int group, int table_width, int pages, int page_size,
                                void* workspace, size_t workspace_bytes, void* stream)
{
    if (rows <= 0) return FORGE_OK;
    if (rows > kForkRows || group <= 0 || rows % group != 0 || table_width <= 0 || pages <= 0 || page_size <= 0 ||
        (page_size & (page_size - 1)) != 0 || static_cast<long long>(pages) * page_size > INT_MAX + 1LL ||
        static_cast<long long>(table_width) * page_size > INT_MAX || !page_table || !cache_lens || !parents || !refs || !table_out ||
        !lens_out || !refs_out || !slots || !src || !dst || !workspace || !aligned(workspace, 4) ||
        workspace_bytes < forge_fork_pages_workspace_size(rows, pages))
        return FORGE_EINVAL;
    // the second launch reads what the outputs would overwrite
    const size_t table = static_cast<size_t>(rows) * table_width;
    if (overlap(page_table, table, table_out, table) || overlap(refs, pages, refs_out, pages) || overlap(cache_lens, rows, lens_out, rows))
        return FORGE_EINVAL;
    int32_t* rank = static_cast<int32_t*>(workspace);
    const ForkArgs a{page_table, cache_lens, parents, refs, table_out, lens_out, refs_out, slots, src, dst, rank, rank + rows,
                     rows, group, table_width, pages, __builtin_ctz(static_cast<unsigned>(page_size))};
    hipStream_t s = as_stream(stream);
    fork_rows_kernel<<<static_cast<unsigned>(1 + divup(pages, kForkPart)), kForkThreads, 4 * rows, s>>>(a);
    const int st = launch_status();
    if (st != FORGE_OK) return st;
    fork_table_kernel<<<static_cast<unsigned>(rows), kForkThreads, 0, s>>>(a);
    return launch_status();
}

extern "C" int forge_copy_pages(void* const* caches, int tensors, long long page_bytes, int pages, const int32_t* src,
                                const int32_t* dst, int pairs, void* stream)
{
    if (tensors <= 0 || pairs <= 0 || page_bytes <= 0) return FORGE_OK;
    if (!caches || !src || !dst || pages <= 0 || page_bytes % 16 != 0 || page_bytes > (1LL << 40)) return FORGE_EINVAL;
    for (int i = 0; i < tensors; i++)
        if (!caches[i] || !aligned(caches[i], 16)) return FORGE_EINVAL;
    hipStream_t s = as_stream(stream);
    CopyArgs a{};
    a.src = src;
    a.dst = dst;
    a.page_bytes = page_bytes;
    a.pairs = pairs;
    a.pages = pages;
    for (int t = 0; t < tensors; t += kCopyTensors) {
        const int n = std::min(kCopyTensors, tensors - t);
        for (int i = 0; i < n; i++) a.tensor[i] = static_cast<uint8_t*>(caches[t + i]);
        const dim3 grid(static_cast<unsigned>(divupll(page_bytes, 4096)), static_cast<unsigned>(std::min(pairs, 65535)), static_cast<unsigned>(n));
        copy_pages_kernel<<<grid, 256, 0, s>>>(a);
        const int st = launch_status();
        if (st != FORGE_OK) return st;
    }
    return FORGE_OK;
}
