// A beam search's next tokens: of the W beams of each request, score[w, v] = logit[w, v] - logsumexp(logit[w]) + score[w],
// the `count` largest of all W x V, ties to the lowest (w, v).
//
// Bound: reading the logits once. A workgroup takes a piece of one row into registers: the piece's maximum and sum of
// exponentials, and its `count` largest logits. Within a row the order is the logits' own, so no sum is needed for that. The pieces' lists
// are merged by a workgroup per request, in 64 bits: the scores of two beams may differ in the last place only.
//
// The largest of n numbers with a total order (value, then lowest place): 64 groups' maxima are ranked, the count-th of them is a bound that at
// least `count` numbers reach, and what reaches it, few more as a rule, is gathered in LDS and ranked by counting.
#include "float16_types.h"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace forge_amd {

constexpr int kBeamCount = 64;      // places
constexpr int kBeamWidth = 1024;    // beams of a request
constexpr int kBeamRoom = 1024;     // numbers that are ranked at once
constexpr int kBeamThreads = 256;

struct BeamPiece {       // of a row: its largest logit and sum of exp(logit - largest)
    double sum;
    float top, unused;
};
struct BeamEntry {
    float logit;
    int token;           // -1: none
};

struct BeamArgs {
    const void* logits;
    const float* scores;
    const uint8_t* ended;
    float* out_scores;
    int32_t *out_beams, *out_tokens;
    BeamPiece* pieces;
    BeamEntry* entries;
    long long batch_stride, beam_stride;
    int B, W, V, count, end_token, splits;
};

// Logits as keys that order as (value, lowest place); 0 for -inf, which no place takes.
template <class T>
struct Logits16 {
    typedef uint16_t Elem;
    typedef uint32_t Key;
    static constexpr int kPer = 8;
    static __device__ __forceinline__ float value(const v4u& v, int e) {
        return T::widen(static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1))));
    }
    static __device__ __forceinline__ Key key(const v4u& v, int e, int place) {
        uint32_t h = v[e / 2] >> (16 * (e & 1)) & 0xFFFFu;
        h = h == 0x8000u ? 0u : h;                                   // -0 is 0
        const uint32_t o = h & 0x8000u ? h ^ 0xFFFFu : h | 0x8000u;
        return o > (T::kInfinity ^ 0x7FFFu) ? o << 16 | (0xFFFFu - place) : 0u;
    }
    static __device__ __forceinline__ int place(Key k) { return static_cast<int>(0xFFFFu - (k & 0xFFFFu)); }
    static __device__ __forceinline__ float of(Key k) {
        const uint32_t o = k >> 16;
        return T::widen(static_cast<uint16_t>(o & 0x8000u ? o ^ 0x8000u : o ^ 0xFFFFu));
    }
    static __device__ __forceinline__ v4u nothing() { return v4u{1u, 1u, 1u, 1u} * (0x80008000u | T::kInfinity * 0x10001u); }
};
struct Logits32 {
    typedef float Elem;
    typedef unsigned long long Key;
    static constexpr int kPer = 4;
    static __device__ __forceinline__ float value(const v4u& v, int e) { return __uint_as_float(v[e]); }
    static __device__ __forceinline__ Key key(const v4u& v, int e, int place) {
        uint32_t h = v[e];
        h = h == 0x80000000u ? 0u : h;
        const uint32_t o = h & 0x80000000u ? ~h : h | 0x80000000u;
        return o > 0x007FFFFFu ? static_cast<Key>(o) << 32 | (0xFFFFFFFFu - place) : 0u;
    }
    static __device__ __forceinline__ int place(Key k) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k)); }
    static __device__ __forceinline__ float of(Key k) {
        const uint32_t o = static_cast<uint32_t>(k >> 32);
        return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
    }
    static __device__ __forceinline__ v4u nothing() { return v4u{1u, 1u, 1u, 1u} * 0xFF800000u; }
};

template <class K>
__device__ __forceinline__ K lane_value(K x, int lane) {
    if constexpr (sizeof(K) == 4) {
        return static_cast<K>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
    } else {
        uint64_t u = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
        return __builtin_bit_cast(K, static_cast<uint64_t>(hi) << 32 | lo);
    }
}

template <class K> __device__ __forceinline__ K highest() { return ~K(0); }
template <> __device__ __forceinline__ double highest<double>() { return INFINITY; }

// The nth largest (from 0) of a wave's 64 keys; equal ones count once each.
template <class K>
__device__ __forceinline__ K wave_nth(K x, int n) {
    int above = 0;
#pragma unroll
    for (int l = 0; l < kWave; l++) above += lane_value(x, l) > x;
    // the smallest of those that n or fewer are above
    K least = above <= n ? x : highest<K>();
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const K y = static_cast<K>(__shfl_xor(least, o, kWave));
        least = y < least ? y : least;
    }
    return least;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) x += __shfl_xor(x, o, kWave);
    return x;
}
// A row's piece of 256 x VEC vectors of 16 bytes. Places are counted from the piece's start, whatever its address, so that equal rows
// have equal sums.
template <class L, int VEC>
__global__ __launch_bounds__(kBeamThreads) void beam_piece_kernel(BeamArgs a)
{
    typedef typename L::Key Key;
    constexpr int kPiece = kBeamThreads * VEC * L::kPer;
    __shared__ Key group[4][kWave];
    __shared__ Key found[kBeamRoom];
    __shared__ double part_sum[4];
    __shared__ float part_top[4];
    __shared__ Key part_key[4];
    __shared__ int total;

    const unsigned row = blockIdx.x / static_cast<unsigned>(a.splits), split = blockIdx.x - row * a.splits;
    if (a.ended && a.ended[row]) return;                             // its one candidate needs no logits
    const unsigned batch = row / static_cast<unsigned>(a.W), beam = row - batch * a.W;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int first = split * kPiece, n = min(a.V - first, kPiece);
    const typename L::Elem* p = static_cast<const typename L::Elem*>(a.logits) + batch * a.batch_stride + beam * a.beam_stride + first;

    typedef v4u loose __attribute__((aligned(2)));
    v4u v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        const int at = (i * kBeamThreads + tid) * L::kPer;
        v[i] = L::nothing();
        if (at + L::kPer <= n) {
            v[i] = *reinterpret_cast<const loose*>(p + at);
        } else if (at < n) {
#pragma unroll
            for (int e = 0; e < L::kPer; e++) {
                if (at + e >= n) continue;
                if constexpr (L::kPer == 8) {
                    const uint32_t h = p[at + e];
                    v[i][e / 2] = e & 1 ? (v[i][e / 2] & 0xFFFFu) | h << 16 : (v[i][e / 2] & 0xFFFF0000u) | h;
                } else {
                    v[i][e] = __float_as_uint(p[at + e]);
                }
            }
        }
    }

    float top = -FLT_MAX;
    Key best = 0;
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (int e = 0; e < L::kPer; e++) {
            top = fmaxf(top, L::value(v[i], e));
            best = max(best, L::key(v[i], e, (i * kBeamThreads + tid) * L::kPer + e));
        }
    top = wave_max(top);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (int e = 0; e < L::kPer; e++) sum += __builtin_amdgcn_exp2f((L::value(v[i], e) - top) * 1.44269504f);
    const double wsum = wave_sum(sum);
    if (lane == 0) {
        part_top[wave] = top;
        part_sum[wave] = wsum;
    }
    if (tid == 0) total = 0;
    group[wave][lane] = best;
    __syncthreads();
    if (tid == 0) {
        const float m = fmaxf(fmaxf(part_top[0], part_top[1]), fmaxf(part_top[2], part_top[3]));
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < 4; w++) s += part_sum[w] * exp(static_cast<double>(part_top[w]) - m);
        a.pieces[static_cast<size_t>(row) * a.splits + split] = {s, m, 0.0f};
    }
    const Key bound = max(wave_nth(max(max(group[0][lane], group[1][lane]), max(group[2][lane], group[3][lane])), a.count - 1), Key(1));
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (int e = 0; e < L::kPer; e++) {
            const Key k = L::key(v[i], e, (i * kBeamThreads + tid) * L::kPer + e);
            if (k >= bound) {
                const int at = atomicAdd(&total, 1);
                if (at < kBeamRoom) found[at] = k;
            }
        }
    __syncthreads();
    BeamEntry* out = a.entries + (static_cast<size_t>(row) * a.splits + split) * a.count;
    auto put = [&](int place, Key k) { out[place] = k ? BeamEntry{L::of(k), first + L::place(k)} : BeamEntry{0.0f, -1}; };
    const int got = total;
    if (got <= kBeamRoom) {
        for (int i = tid; i < got; i += kBeamThreads) {
            const Key k = found[i];
            int rank = 0;
            for (int j = 0; j < got; j++) rank += found[j] > k;
            if (rank < a.count) put(rank, k);
        }
        for (int i = got + tid; i < a.count; i += kBeamThreads) put(i, 0);
        return;
    }
    // more than there is room for (long runs of large neighbours): one place after the other
    Key last = ~Key(0);
    for (int place = 0; place < a.count; place++) {
        Key next = 0;
#pragma unroll
        for (int i = 0; i < VEC; i++)
#pragma unroll
            for (int e = 0; e < L::kPer; e++) {
                const Key k = L::key(v[i], e, (i * kBeamThreads + tid) * L::kPer + e);
                if (k < last && k > next) next = k;
            }
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) next = max(next, static_cast<Key>(__shfl_xor(next, o, kWave)));
        if (lane == 0) part_key[wave] = next;
        __syncthreads();
        last = max(max(part_key[0], part_key[1]), max(part_key[2], part_key[3]));
        __syncthreads();
        if (tid == 0) put(place, last);
        if (last == 0) last = 1;                                     // nothing is left: no key is below 1
    }
}

// The candidates of a request: entry i of the pieces' lists, then one per beam that has ended.
struct BeamCandidate {
    double score;
    unsigned long long place;    // beam * 2^32 + token
};
__device__ __forceinline__ bool beam_before(const BeamCandidate& x, const BeamCandidate& y) {
    return x.score > y.score || (x.score == y.score && x.place < y.place);
}

__global__ __launch_bounds__(kBeamThreads) void beam_merge_kernel(BeamArgs a)
{
    __shared__ double shift[kBeamWidth];     // score - logsumexp, -inf for a beam without candidates
    __shared__ double group[4][kWave];
    __shared__ BeamCandidate found[kBeamRoom];
    __shared__ BeamCandidate part[4];
    __shared__ int total;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const size_t row0 = static_cast<size_t>(blockIdx.x) * a.W;
    for (int w = wave; w < a.W; w += 4) {
        const size_t row = row0 + w;
        const bool ended = a.ended && a.ended[row];
        const BeamPiece* p = a.pieces + row * a.splits;
        float top = -FLT_MAX;
        double sum = 0.0;
        if (!ended) {
            for (int i = lane; i < a.splits; i += kWave) top = fmaxf(top, p[i].top);
            top = wave_max(top);
            for (int i = lane; i < a.splits; i += kWave) sum += p[i].sum * exp(static_cast<double>(p[i].top) - top);
            sum = wave_sum(sum);
        }
        const double score = a.scores[row];
        // rows with an infinity or NaN have no sum, and rows of -inf only a sum of zero
        const bool live = ended || (sum > 0.0 && sum < INFINITY && top < INFINITY);
        if (lane == 0) shift[w] = live && fabs(score) < INFINITY ? (ended ? score : score - (top + log(sum))) : -INFINITY;
    }
    if (tid == 0) total = 0;
    __syncthreads();
    const int per = a.splits * a.count, lists = a.W * per;           // (below 2^31: the launcher's check)
    auto candidate = [&](int i) -> BeamCandidate {
        if (i >= lists) {
            const int w = i - lists;
            return {a.ended && a.ended[row0 + w] ? shift[w] : -INFINITY,
                    static_cast<unsigned long long>(w) << 32 | static_cast<uint32_t>(a.end_token)};
        }
        const int w = static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(per));
        if (shift[w] == -INFINITY || (a.ended && a.ended[row0 + w])) return {-INFINITY, 0ull};
        const BeamEntry e = a.entries[row0 * per + i];
        return {e.token < 0 ? -INFINITY : e.logit + shift[w], static_cast<unsigned long long>(w) << 32 | static_cast<uint32_t>(e.token)};
    };
    const int all = lists + (a.ended ? a.W : 0);
    double best = -INFINITY;
    for (int i = tid; i < all; i += kBeamThreads) best = fmax(best, candidate(i).score);
    group[wave][lane] = best;
    __syncthreads();
    const double bound = wave_nth(fmax(fmax(group[0][lane], group[1][lane]), fmax(group[2][lane], group[3][lane])), a.count - 1);
    for (int i = tid; i < all; i += kBeamThreads) {
        const BeamCandidate c = candidate(i);
        if (c.score > -INFINITY && c.score >= bound) {
            const int at = atomicAdd(&total, 1);
            if (at < kBeamRoom) found[at] = c;
        }
    }
    __syncthreads();
    const size_t out = static_cast<size_t>(blockIdx.x) * a.count;
    auto put = [&](int place, const BeamCandidate& c) {
        const bool some = c.score > -INFINITY;
        a.out_scores[out + place] = some ? static_cast<float>(c.score) : -INFINITY;
        a.out_beams[out + place] = some ? static_cast<int>(c.place >> 32) : -1;
        a.out_tokens[out + place] = some ? static_cast<int>(c.place & 0xFFFFFFFFu) : -1;
    };
    const BeamCandidate none = {-INFINITY, ~0ull};
    const int got = total;
    if (got <= kBeamRoom) {
        for (int i = tid; i < got; i += kBeamThreads) {
            const BeamCandidate c = found[i];
            int rank = 0;
            for (int j = 0; j < got; j++) rank += beam_before(found[j], c);
            if (rank < a.count) put(rank, c);
        }
        for (int i = got + tid; i < a.count; i += kBeamThreads) put(i, none);
        return;
    }
    BeamCandidate last = {INFINITY, 0ull};
    for (int place = 0; place < a.count; place++) {                  // one place after the other
        BeamCandidate next = none;
        for (int i = tid; i < all; i += kBeamThreads) {
            const BeamCandidate c = candidate(i);
            if (c.score > -INFINITY && beam_before(last, c) && beam_before(c, next)) next = c;
        }
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const BeamCandidate c = {__shfl_xor(next.score, o, kWave), static_cast<unsigned long long>(__shfl_xor(next.place, o, kWave))};
            if (beam_before(c, next)) next = c;
        }
        if (lane == 0) part[wave] = next;
        __syncthreads();
        last = part[0];
#pragma unroll
        for (int w = 1; w < 4; w++)
            if (beam_before(part[w], last)) last = part[w];
        __syncthreads();
        if (tid == 0) put(place, last);
    }
}

// Vectors of a thread: 4, or 1 while that leaves CUs without work.
inline int beam_vectors(int B, int W, int V, int per) {
    return static_cast<long long>(B) * W * divup(V, kBeamThreads * 4 * per) >= 2 * default_cu_count() ? 4 : 1;
}
inline bool beam_shape_ok(int B, int W, int V, int count) {
    return B > 0 && W > 0 && W <= kBeamWidth && V > 0 && count > 0 && count <= kBeamCount &&
           static_cast<long long>(B) * W * divup(V, kBeamThreads * 4) <= INT_MAX &&
           static_cast<long long>(W) * (divup(V, kBeamThreads * 4) * static_cast<long long>(count) + 1) <= INT_MAX - kBeamThreads;
}
inline int beam_per(int dtype) { return dtype == FORGE_FP32 ? 4 : 8; }
inline size_t beam_bytes(int B, int W, int count, int splits) {
    return static_cast<size_t>(B) * W * splits * (sizeof(BeamPiece) + count * sizeof(BeamEntry));
}

template <class L>
int launch_beams(const BeamArgs& a, int vectors, hipStream_t s) {
    const unsigned grid = static_cast<unsigned>(a.B) * a.W * a.splits;
    if (vectors == 4) beam_piece_kernel<L, 4><<<grid, kBeamThreads, 0, s>>>(a);
    else beam_piece_kernel<L, 1><<<grid, kBeamThreads, 0, s>>>(a);
    const int st = launch_status();
    if (st != FORGE_OK) return st;
    beam_merge_kernel<<<static_cast<unsigned>(a.B), kBeamThreads, 0, s>>>(a);
    return launch_status();
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_beam_select_workspace_size(int B, int W, int V, int count) {
    if (!beam_shape_ok(B, W, V, count)) return 0;
    size_t most = 0;                                                 // of any type
    for (int per : {4, 8}) most = std::max(most, beam_bytes(B, W, count, divup(V, kBeamThreads * beam_vectors(B, W, V, per) * per)));
    return most;
}

extern "C" int forge_beam_select(const void* logits, const float* scores, const uint8_t* ended, int end_token, float* out_scores,
                                 int32_t* out_beams, int32_t* out_tokens, int B, int W, int V, int count,
                                 long long batch_stride, long long beam_stride, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    if (B <= 0 || W <= 0 || V <= 0 || count <= 0) return FORGE_OK;
    if (!beam_shape_ok(B, W, V, count) || !logits || !scores || !out_scores || !out_beams || !out_tokens || batch_stride < 0 ||
        beam_stride < 0 || (dtype != FORGE_FP16 && dtype != FORGE_BF16 && dtype != FORGE_FP32) ||
        (ended && (end_token < 0 || end_token >= V)) || !aligned(logits, dtype == FORGE_FP32 ? 4 : 2))
        return FORGE_EINVAL;
    const int per = beam_per(dtype), vectors = beam_vectors(B, W, V, per), splits = divup(V, kBeamThreads * vectors * per);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < beam_bytes(B, W, count, splits)) return FORGE_EINVAL;
    BeamPiece* pieces = static_cast<BeamPiece*>(workspace);
    const BeamArgs a{logits, scores, ended, out_scores, out_beams, out_tokens, pieces,
                     reinterpret_cast<BeamEntry*>(pieces + static_cast<size_t>(B) * W * splits), batch_stride, beam_stride,
                     B, W, V, count, end_token, splits};
    hipStream_t s = as_stream(stream);
    if (dtype == FORGE_FP32) return launch_beams<Logits32>(a, vectors, s);
    return dtype == FORGE_FP16 ? launch_beams<Logits16<Fp16>>(a, vectors, s) : launch_beams<Logits16<Bf16>>(a, vectors, s);
}
