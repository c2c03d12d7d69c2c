// The pages of a paged cache whose rows go on from one another, as a beam search's do after a selection.
//
// fork_pages: new row r goes on from row p of its group, parents[r] of it (none: the row ends). It names p's full pages again, without a copy;
// refs counts the names of each page. The page of its next token is p's own where p's first child takes it and nobody else
// names it, else the lowest free page not yet taken, the next for each row in order; the filled part of p's page is then to be copied (src, dst). Pages that
// this call frees are not taken by it, so no copied page is written. A row without a free page to copy into has lost the tokens of that page, which
// its entry of -1 beside a length inside the page says to the next call: rows that would go on from it end there, since the page that they would
// get is new, or was another row's. Counts are added to with integer atomics, whose order does not matter; everything else is in the rows' order.
//
// Bound: latency. Small tables and pools take one workgroup that holds all counts in LDS (4 rows of 40 entries 3.7 us), others two launches:
// first, a workgroup looks at the rows (first children, places among the takers) while others copy the counts and list the free pages of 1024 pages
// each; then a workgroup per row finds its page and writes its table (512 rows of 128 entries, 4000 pages, 3.9 + 3.6 us). copy_pages: memory; 8 tensors
// of 16 KB pages, some 300 pairs, 10.8 us.
#include "common.h"

#include <algorithm>
#include <climits>

namespace forge_amd {

constexpr int kForkRows = 8192;      // rows that one workgroup looks at (first children in LDS)
constexpr int kForkThreads = 1024, kTableThreads = 256;
constexpr int kForkPart = 1024;      // pages whose free ones are listed together

struct ForkRow {
    int parent, len, last;   // parent: -1 none; last: its page of the next token, or -1
    int rank;                // the row's place among those that take a page, or -1
};
struct ForkArgs {
    const int32_t *table, *lens, *parents, *refs;
    int32_t *table_out, *lens_out, *refs_out, *slots, *src, *dst;
    ForkRow* row;
    int32_t *counts, *free;  // free pages of each part, and their numbers (kForkPart places a part)
    int rows, group, width, pages, page_shift;
};

// Sum over the threads before this one, and over all (in *all), of a workgroup of N.
template <int N>
__device__ __forceinline__ int sum_before(int x, int* all, int (&part)[N / kWave]) {
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
    *all = 0;
#pragma unroll
    for (int w = 0; w < N / kWave; w++) {
        before += w < wave ? part[w] : 0;
        *all += part[w];
    }
    return before;
}

// Row r as its parent leaves it, but for its rank.
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int parent) {
    ForkRow row = {parent, 0, -1, -1};
    if (parent < 0) return row;
    row.len = min(max(a.lens[parent], 0), a.width << a.page_shift);
    const int at = row.len >> a.page_shift;
    const int pg = at < a.width ? a.table[static_cast<size_t>(parent) * a.width + at] : -1;
    row.last = pg >= 0 && pg < a.pages ? pg : -1;
    const bool lost = pg < 0 && (row.len & ((1 << a.page_shift) - 1)) != 0;
    row.parent = lost ? -1 : parent;
    row.len = lost ? 0 : row.len;
    return row;
}
__device__ __forceinline__ int fork_parent(const ForkArgs& a, int r) {
    const int p = a.parents[r];
    return p >= 0 && p < a.group ? r - r % a.group + p : -1;
}
__device__ __forceinline__ void fork_put(const ForkArgs& a, int r, const ForkRow& row, int page) {
    const int in_page = row.len & ((1 << a.page_shift) - 1);
    const bool copied = row.rank >= 0 && page >= 0 && row.last >= 0 && in_page > 0;
    a.lens_out[r] = row.len;
    a.slots[r] = page >= 0 ? (page << a.page_shift) + in_page : -1;
    a.src[r] = copied ? row.last : -1;
    a.dst[r] = copied ? page : -1;
}

// All of it in one workgroup. us in a graph, this and the two launches: 4 rows of 40 entries and 59 pages 4.1 and 5.3, 128 of 32 and 1061
// 5.6 and 6.1, 128 of 128 9.8 and 6.1, 512 of 16 and 3461 8.0 and 6.5.
constexpr int kSmallRows = 1024, kSmallPages = 2048, kSmallTable = 4096;
__global__ __launch_bounds__(kForkThreads) void fork_small_kernel(ForkArgs a)
{
    __shared__ int counts[kSmallPages], first[kSmallRows], free[kSmallRows], mine[kSmallRows], up[kSmallRows], from[kSmallRows];
    __shared__ int part[kForkThreads / kWave];
    const int tid = threadIdx.x;
    int p = -1, x[kSmallPages / kForkThreads], all;
#pragma unroll
    for (int i = 0; i < kSmallPages / kForkThreads; i++) {
        const int pg = tid + i * kForkThreads;
        x[i] = pg < a.pages ? a.refs[pg] : 1;
    }
    if (tid < a.rows) {
        first[tid] = a.rows;
        p = fork_parent(a, tid);
    }
    __syncthreads();
    if (p >= 0) atomicMin(&first[p], tid);
    ForkRow row = fork_row(a, p);
    p = row.parent;
    int base = 0;                                                    // the lowest free pages, one a row at most
#pragma unroll
    for (int i = 0; i < kSmallPages / kForkThreads; i++) {
        const int pg = tid + i * kForkThreads;
        counts[pg] = x[i];
        if (i * kForkThreads >= a.pages || base >= a.rows) continue;
        const int before = base + sum_before<kForkThreads>(x[i] == 0, &all, part);
        if (x[i] == 0 && before < a.rows) free[before] = pg;
        base += all;
    }
    __syncthreads();
    const int at = row.len >> a.page_shift;
    const bool take = p >= 0 && at < a.width && !(row.last >= 0 && first[p] == tid && counts[row.last] == 1);
    const int rank = sum_before<kForkThreads>(take, &all, part);
    if (tid < a.rows) {
        if (take) row.rank = rank;
        const int page = !take ? row.last : rank < base ? free[rank] : -1;
        mine[tid] = page;
        up[tid] = p;
        from[tid] = at;
        fork_put(a, tid, row, page);
    }
    __syncthreads();
    for (int i = tid; i < a.rows * a.width; i += kForkThreads) {
        const int r = static_cast<unsigned>(i) / static_cast<unsigned>(a.width), c = i - r * a.width, q = up[r];
        const int old = a.table[i];
        int pg = q >= 0 && c < from[r] ? a.table[q * a.width + c] : c == from[r] ? mine[r] : -1;
        if (pg < 0 || pg >= a.pages) pg = -1;
        a.table_out[i] = pg;
        if (old != pg) {
            if (old >= 0 && old < a.pages) atomicAdd(&counts[old], -1);
            if (pg >= 0) atomicAdd(&counts[pg], 1);
        }
    }
    __syncthreads();
    for (int pg = tid; pg < a.pages; pg += kForkThreads) a.refs_out[pg] = counts[pg];
}

__global__ __launch_bounds__(kForkThreads) void fork_rows_kernel(ForkArgs a)
{
    __shared__ int part[kForkThreads / kWave];
    const int tid = threadIdx.x;
    int all;
    if (blockIdx.x > 0) {                                            // a part of the counts
        const int which = blockIdx.x - 1, pg = which * kForkPart + tid;
        const int x = pg < a.pages ? a.refs[pg] : 1;
        if (pg < a.pages) a.refs_out[pg] = x;
        const int before = sum_before<kForkThreads>(x == 0, &all, part);
        if (x == 0) a.free[which * kForkPart + before] = pg;
        if (tid == 0) a.counts[which] = all;
        return;
    }
    extern __shared__ int first[];                                   // a row's first child
    for (int r = tid; r < a.rows; r += kForkThreads) first[r] = a.rows;
    __syncthreads();
    for (int r = tid; r < a.rows; r += kForkThreads) {
        const int p = fork_parent(a, r);
        if (p >= 0) atomicMin(&first[p], r);
    }
    __syncthreads();
    int base = 0;
    for (int r0 = 0; r0 < a.rows; r0 += kForkThreads) {
        const int r = r0 + tid;
        ForkRow row = {-1, 0, -1, -1};
        bool take = false;
        if (r < a.rows) {
            const int p = fork_parent(a, r);
            row = fork_row(a, p);
            const int names = a.refs[max(row.last, 0)], child = first[max(p, 0)];   // (at once, with no branch between)
            take = row.parent >= 0 && row.len >> a.page_shift < a.width && !(row.last >= 0 && child == r && names == 1);
        }
        const int before = sum_before<kForkThreads>(take, &all, part);
        if (take) row.rank = base + before;
        if (r < a.rows) a.row[r] = row;
        base += all;
    }
}

__global__ __launch_bounds__(kTableThreads) void fork_table_kernel(ForkArgs a)
{
    __shared__ int part[kTableThreads / kWave], mine;
    const int r = blockIdx.x, tid = threadIdx.x;
    const ForkRow row = a.row[r];
    const int at = row.len >> a.page_shift, p = row.parent;
    const int32_t* from = a.table + static_cast<size_t>(max(p, 0)) * a.width;
    const int32_t* was = a.table + static_cast<size_t>(r) * a.width;
    int32_t* to = a.table_out + static_cast<size_t>(r) * a.width;
    // (loaded before the search for a page)
    const int i0 = min(tid, a.width - 1), from0 = from[i0], was0 = was[i0];
    int page = row.rank < 0 ? row.last : -1;
    if (row.rank >= 0) {
        // the part that has the rank-th free page
        if (tid == 0) mine = -1;
        const int parts = (a.pages + kForkPart - 1) / kForkPart;
        int left = row.rank;
        for (int j = 0; j < parts; j += kTableThreads) {
            const int x = j + tid < parts ? a.counts[j + tid] : 0;
            int all;
            const int before = sum_before<kTableThreads>(x, &all, part);
            if (before <= left && left < before + x) mine = a.free[(j + tid) * kForkPart + left - before];
            if (left < all) break;
            left -= all;
        }
        __syncthreads();
        page = mine;
    }
    if (tid == 0) fork_put(a, r, row, page);
    // the old row's names go, the new row's come
    for (int i = tid; i < a.width; i += kTableThreads) {
        const int old = i == tid ? was0 : was[i];
        int pg = p >= 0 && i < at ? (i == tid ? from0 : from[i]) : i == at ? page : -1;
        if (pg < 0 || pg >= a.pages) pg = -1;
        to[i] = pg;
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
    long long page_bytes, left;   // left: of a page, from the tensors' addresses on
    int pairs, pages;
};

// A workgroup copies 4 KB of one page: blockIdx.x the piece, y the pair, z the tensor.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a)
{
    for (int i = blockIdx.y; i < a.pairs; i += gridDim.y) {
        const int s = a.src[i], d = a.dst[i];
        if (s < 0 || d < 0 || s >= a.pages || d >= a.pages || s == d) continue;
        const long long at = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 16;
        if (at >= a.left) continue;
        uint8_t* t = a.tensor[blockIdx.z];
        *reinterpret_cast<uint4*>(t + d * a.page_bytes + at) = *reinterpret_cast<const uint4*>(t + s * a.page_bytes + at);
    }
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_fork_pages_workspace_size(int rows, int pages) {
    if (rows <= 0 || rows > kForkRows || pages <= 0) return 0;
    const size_t parts = divup(pages, kForkPart);
    return sizeof(ForkRow) * rows + 4 * parts * (1 + kForkPart);
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
        !lens_out || !refs_out || !slots || !src || !dst || !workspace || !aligned(workspace, 16) ||
        workspace_bytes < forge_fork_pages_workspace_size(rows, pages))
        return FORGE_EINVAL;
    // the second launch reads what the outputs would overwrite
    const size_t table = static_cast<size_t>(rows) * table_width;
    if (overlap(page_table, table, table_out, table) || overlap(refs, pages, refs_out, pages) || overlap(cache_lens, rows, lens_out, rows))
        return FORGE_EINVAL;
    const int parts = divup(pages, kForkPart);
    ForkRow* row = static_cast<ForkRow*>(workspace);
    int32_t* counts = reinterpret_cast<int32_t*>(row + rows);
    const ForkArgs a{page_table, cache_lens, parents, refs, table_out, lens_out, refs_out, slots, src, dst, row, counts, counts + parts,
                     rows, group, table_width, pages, __builtin_ctz(static_cast<unsigned>(page_size))};
    hipStream_t s = as_stream(stream);
    if (rows <= kSmallRows && pages <= kSmallPages && table <= kSmallTable) {
        fork_small_kernel<<<1, kForkThreads, 0, s>>>(a);
        return launch_status();
    }
    fork_rows_kernel<<<static_cast<unsigned>(1 + parts), kForkThreads, 4 * rows, s>>>(a);
    const int st = launch_status();
    if (st != FORGE_OK) return st;
    fork_table_kernel<<<static_cast<unsigned>(rows), kTableThreads, 0, s>>>(a);
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
    const long long most = grid_limit(256) * 4096;                   // of a page, by a launch
    for (int t = 0; t < tensors; t += kCopyTensors) {
        const int n = std::min(kCopyTensors, tensors - t);
        for (long long at = 0; at < page_bytes; at += most) {
            for (int i = 0; i < n; i++) a.tensor[i] = static_cast<uint8_t*>(caches[t + i]) + at;
            a.left = page_bytes - at;
            const dim3 grid(static_cast<unsigned>(divupll(std::min(a.left, most), 4096)), static_cast<unsigned>(std::min(pairs, 65535)),
                            static_cast<unsigned>(n));
            copy_pages_kernel<<<grid, 256, 0, s>>>(a);
            const int st = launch_status();
            if (st != FORGE_OK) return st;
        }
    }
    return FORGE_OK;
}
