// A beam search's next tokens: of the W beams of each request, score[w, v] = logit[w, v] - logsumexp(logit[w]) + score[w],
// the `count` largest of all W x V, ties to the lowest (w, v).
//
// Bound: reading the logits once. A workgroup takes a piece of one row into registers: the piece's maximum and sum of
// exponentials, and its `count` largest logits. Within a row the order is the logits' own, so no sum is needed for that. The pieces' lists
// are merged by a workgroup per request, in 64 bits: the scores of two beams may differ in the last place only.
//
// The largest of many: of 64 groups' maxima the count-th largest is a bound that at least `count` numbers reach, and what reaches it, few
// more as a rule, is gathered in LDS and ranked by counting, with ties by place. Where more are found, a better bound comes from those (most lists
// empty, or many places), or they are equal ones (a mask's lowest value): those above the bound are ranked and the first places that equal
// it follow. Where a piece has more of those than LDS has room, its places are filled one after the other.
//
// us, pieces + merge: 32 x 8 beams of 131072 FP32 logits, three in ten ended, 18.5 (94 MB at 5.1 TB/s) + 8.5; 4 beams of 32000 FP16 4.6 + 5.5, two chains
// of dependent steps. In all, 8 x 4 beams of 128000, 16 places: 15; all but 20 tokens at FP16's lowest value 20 (place after place 65), all logits
// equal 41 (60); 4 x 8 of 50257, 53 places: 25 (ranking all that the first bound leaves 49), one live beam 25 (137), all equal 33 (433).
#include "float16_types.h"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace forge_amd {

constexpr int kBeamCount = 64;      // places
constexpr int kBeamWidth = 1024;    // beams of a request
constexpr int kBeamRoom = 1024;     // numbers that are ranked at once
constexpr int kBeamFew = 256;       // and as many as are ranked without looking for a better bound
constexpr int kBeamThreads = 256, kMergeThreads = 512;

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

// Vectors of 16 bytes of logits.
template <class T>
struct Logits16 {
    typedef uint16_t Elem;
    static constexpr int kPer = 8, kMany = 4;
    static __device__ __forceinline__ float value(const v4u& v, int e) {
        return T::widen(static_cast<uint16_t>(v[e / 2] >> (16 * (e & 1))));
    }
    static __device__ __forceinline__ uint32_t nothing() { return (0x8000u | T::kInfinity) * 0x10001u; }
    static __device__ __forceinline__ void set(v4u& v, int e, Elem x) {
        v[e / 2] = e & 1 ? (v[e / 2] & 0xFFFFu) | static_cast<uint32_t>(x) << 16 : (v[e / 2] & 0xFFFF0000u) | x;
    }
};
struct Logits32 {
    typedef uint32_t Elem;
    static constexpr int kPer = 4, kMany = 8;
    static __device__ __forceinline__ float value(const v4u& v, int e) { return __uint_as_float(v[e]); }
    static __device__ __forceinline__ uint32_t nothing() { return 0xFF800000u; }
    static __device__ __forceinline__ void set(v4u& v, int e, Elem x) { v[e] = x; }
};

// Keys that order as (value, lowest place), and back.
typedef unsigned long long BeamKey;
__device__ __forceinline__ BeamKey beam_key(float x, int place) {
    const uint32_t h = __float_as_uint(x + 0.0f);                    // -0 is 0
    const uint32_t o = h & 0x80000000u ? ~h : h | 0x80000000u;
    return static_cast<BeamKey>(o) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(place));
}
__device__ __forceinline__ int key_place(BeamKey k) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float key_value(BeamKey k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// Reductions over a wave in registers, the same on all lanes: neighbours, pairs, mirrored halves of 8 and 16 lanes, then rows of 16. (Through LDS
// the same took half a microsecond a kernel.)
template <int STEP>
__device__ __forceinline__ uint32_t other_lane(uint32_t x) {
    constexpr int kCtrl = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kCtrl, 0xF, 0xF, false));
}
template <class F>
__device__ __forceinline__ float wave_reduce(float x, const F& f) {
    auto step = [&](uint32_t y) { x = f(x, __uint_as_float(y)); };
    step(other_lane<0>(__float_as_uint(x)));
    step(other_lane<1>(__float_as_uint(x)));
    step(other_lane<2>(__float_as_uint(x)));
    step(other_lane<3>(__float_as_uint(x)));
    const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const v2u q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
template <class F>
__device__ __forceinline__ double wave_reduce(double x, const F& f) {
    auto words = [&](uint32_t* lo, uint32_t* hi) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        *lo = static_cast<uint32_t>(u);
        *hi = static_cast<uint32_t>(u >> 32);
    };
    auto number = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo); };
    uint32_t lo, hi;
    words(&lo, &hi);
    x = f(x, number(other_lane<0>(lo), other_lane<0>(hi)));
    words(&lo, &hi);
    x = f(x, number(other_lane<1>(lo), other_lane<1>(hi)));
    words(&lo, &hi);
    x = f(x, number(other_lane<2>(lo), other_lane<2>(hi)));
    words(&lo, &hi);
    x = f(x, number(other_lane<3>(lo), other_lane<3>(hi)));
    words(&lo, &hi);
    const v2u l16 = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), h16 = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    x = f(number(l16[0], h16[0]), number(l16[1], h16[1]));
    words(&lo, &hi);
    const v2u l32 = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), h32 = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return f(number(l32[0], h32[0]), number(l32[1], h32[1]));
}
__device__ __forceinline__ double wave_sum(double x) {
    return wave_reduce(x, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ float wave_most(float x) {
    return wave_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}

// The nth largest (from 0) of the 64 groups' largest numbers: each thread compares one of them with some others, the first wave picks the one
// that n are above (the smallest of those that n or fewer are above, where some are equal). All of N threads call it; part[w][l] is
// wave w's largest of group l; the result is wave 0's.
template <class F, int N>
struct NthGroup {
    F part[N / kWave][kWave], group[kWave];
    int above[kWave];
    __device__ __forceinline__ F nth(int n) {
        constexpr int kWaves = N / kWave, kEach = kWave / kWaves;
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
        __syncthreads();
        F x = part[0][lane];
#pragma unroll
        for (int w = 1; w < kWaves; w++) x = x > part[w][lane] ? x : part[w][lane];
        if (wave == 0) {
            group[lane] = x;
            above[lane] = 0;
        }
        __syncthreads();
        int count = 0;
#pragma unroll
        for (int e = 0; e < kEach; e++) count += group[wave * kEach + e] > x;
        atomicAdd(&above[lane], count);
        __syncthreads();
        if (wave != 0) return x;
        const int all = above[lane];
        const unsigned long long at = __ballot(all == n);
        F least = all <= n ? x : static_cast<F>(INFINITY);
        if (at) return __shfl(x, __builtin_ctzll(at), kWave);
        return wave_reduce(least, [](F a, F b) { return b < a ? b : a; });
    }
};

// A row's piece of 256 x VEC vectors. Places are counted from the piece's start, whatever its address, so that equal rows
// have equal sums.
template <class L, int VEC>
__global__ __launch_bounds__(kBeamThreads) void beam_piece_kernel(BeamArgs a)
{
    constexpr int kPiece = kBeamThreads * VEC * L::kPer;
    __shared__ NthGroup<float, kBeamThreads> groups;
    __shared__ BeamKey found[kBeamRoom];
    __shared__ double part_sum[4];
    __shared__ float part_top[4], bound_of;
    __shared__ BeamKey part_key[4];
    __shared__ int total, part_count[2][4];

    const unsigned row = blockIdx.x / static_cast<unsigned>(a.splits), split = blockIdx.x - row * a.splits;
    if (a.ended && a.ended[row]) return;                             // its one candidate needs no logits
    const unsigned batch = row / static_cast<unsigned>(a.W), beam = row - batch * a.W;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int first = split * kPiece, n = min(a.V - first, kPiece);
    const typename L::Elem* p = static_cast<const typename L::Elem*>(a.logits) + batch * a.batch_stride + beam * a.beam_stride + first;

    typedef v4u loose __attribute__((aligned(2)));
    auto load = [&](int i) {
        const int at = (i * kBeamThreads + tid) * L::kPer;
        v4u x = v4u{1u, 1u, 1u, 1u} * L::nothing();
        if (at + L::kPer <= n) {
            x = *reinterpret_cast<const loose*>(p + at);
        } else if (at < n) {
#pragma unroll
            for (int e = 0; e < L::kPer; e++)
                if (at + e < n) L::set(x, e, p[at + e]);
        }
        return x;
    };
    v4u v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = load(i);

    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < VEC; i++)
#pragma unroll
        for (int e = 0; e < L::kPer; e++) most = fmaxf(most, L::value(v[i], e));
    groups.part[wave][lane] = most;
    const float top = fmaxf(wave_most(most), -FLT_MAX);
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
    const float nth = groups.nth(a.count - 1);
    if (tid == 0) {
        bound_of = fmaxf(nth, -FLT_MAX);                             // -inf is no candidate
    } else if (tid == kWave) {
        const float m = fmaxf(fmaxf(part_top[0], part_top[1]), fmaxf(part_top[2], part_top[3]));
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < 4; w++) s += part_sum[w] * exp(static_cast<double>(part_top[w]) - m);
        a.pieces[static_cast<size_t>(row) * a.splits + split] = {s, m, 0.0f};
    }
    __syncthreads();
    const float bound = bound_of;
    auto gather = [&](const v4u& x, int i, auto hit) {
        uint32_t hits = 0u;
#pragma unroll
        for (int e = 0; e < L::kPer; e++) hits |= hit(L::value(x, e)) ? 1u << e : 0u;
        if (!hits) return;
#pragma unroll
        for (int e = 0; e < L::kPer; e++) {
            if (!(hits >> e & 1u)) continue;
            const int at = atomicAdd(&total, 1);
            if (at < kBeamRoom) found[at] = beam_key(L::value(x, e), (i * kBeamThreads + tid) * L::kPer + e);
        }
    };
    BeamEntry* out = a.entries + (static_cast<size_t>(row) * a.splits + split) * a.count;
    auto put = [&](int place, BeamKey k) { out[place] = k ? BeamEntry{key_value(k), first + key_place(k)} : BeamEntry{0.0f, -1}; };
    auto rank = [&](int got) {
        for (int i = tid; i < got; i += kBeamThreads) {
            const BeamKey k = found[i];
            int place = 0;
#pragma unroll 8
            for (int j = 0; j < got; j++) place += found[j] > k;
            if (place < a.count) put(place, k);
        }
    };
    if (most >= bound) {
#pragma unroll
        for (int i = 0; i < VEC; i++) gather(v[i], i, [&](float x) { return x >= bound; });
    }
    __syncthreads();
    int got = total;
    if (got <= 3 * kBeamFew / 2) {
        rank(got);
        for (int i = got + tid; i < a.count; i += kBeamThreads) put(i, 0);
        return;
    }
    // Many, as a rule equal ones (a mask's lowest value): those above the bound, then the first places that equal it. (Loaded again, or the registers
    // would be kept for it.)
    __syncthreads();
    if (tid == 0) total = 0;
    __syncthreads();
    if (most > bound) {
#pragma unroll 1
        for (int i = 0; i < VEC; i++) gather(load(i), i, [&](float x) { return x > bound; });
    }
    __syncthreads();
    got = total;
    if (got <= kBeamRoom) {
        rank(got);
#pragma unroll 1
        for (int i = 0; i < VEC; i++) {
            if (got >= a.count) return;
            const v4u x = load(i);
            int mine = 0;
#pragma unroll
            for (int e = 0; e < L::kPer; e++) mine += L::value(x, e) == bound;
            int place = mine;                                        // of the thread's last one, in its wave
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                const int before = __shfl_up(place, o, kWave);
                place += lane >= o ? before : 0;
            }
            if (lane == kWave - 1) part_count[i & 1][wave] = place;
            __syncthreads();
            place += got - mine;
            for (int w = 0; w < 4; w++) {
                place += w < wave ? part_count[i & 1][w] : 0;
                got += part_count[i & 1][w];
            }
#pragma unroll
            for (int e = 0; e < L::kPer; e++) {
                if (L::value(x, e) != bound) continue;
                if (place < a.count) put(place, beam_key(bound, (i * kBeamThreads + tid) * L::kPer + e));
                place++;
            }
        }
        for (int i = got + tid; i < a.count; i += kBeamThreads) put(i, 0);
        return;
    }
    BeamKey last = ~0ull;
    for (int place = 0; place < a.count; place++) {
        BeamKey next = 0;
#pragma unroll 1
        for (int i = 0; i < VEC; i++) {
            const v4u v_i = load(i);
#pragma unroll
            for (int e = 0; e < L::kPer; e++) {
                const float x = L::value(v_i, e);
                const BeamKey k = beam_key(x, (i * kBeamThreads + tid) * L::kPer + e);
                if (x >= -FLT_MAX && k < last && k > next) next = k;
            }
        }
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) next = max(next, static_cast<BeamKey>(__shfl_xor(next, o, kWave)));
        if (lane == 0) part_key[wave] = next;
        __syncthreads();
        last = max(max(part_key[0], part_key[1]), max(part_key[2], part_key[3]));
        __syncthreads();
        if (tid == 0) put(place, last);                              // (there are more than kBeamRoom)
    }
}

struct BeamCandidate {
    double score;
    unsigned long long place;    // beam * 2^32 + token
};
__device__ __forceinline__ bool beam_before(const BeamCandidate& x, const BeamCandidate& y) {
    return x.score > y.score || (x.score == y.score && x.place < y.place);
}

// A request's candidates: the pieces' lists, each in descending order, and one list of one for each beam that has ended.
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamArgs a)
{
    constexpr int kWaves = kMergeThreads / kWave;
    // a beam's largest logit, and its score - log of the sum of exp(logit - largest), -inf for a beam without candidates (apart, or logits near the
    // type's lowest value would take the score with them)
    __shared__ double shift[kBeamWidth];
    __shared__ float largest[kBeamWidth];
    __shared__ NthGroup<double, kMergeThreads> groups;
    __shared__ BeamCandidate found[kBeamRoom];
    __shared__ int queue[kBeamRoom];
    __shared__ double bound_of;
    __shared__ int total, waiting, part_count[2][kWaves];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const size_t row0 = static_cast<size_t>(blockIdx.x) * a.W;
    const int lists = a.W * a.splits, deep = max(1, min(a.count, kMergeThreads / lists));
    const BeamEntry* entries = a.entries + row0 * a.splits * a.count;
    BeamEntry mine = {0.0f, -1};                                     // (loaded before the sums)
    if (tid < lists * deep) mine = entries[static_cast<size_t>(tid / deep) * a.count + tid % deep];
    for (int w = wave; w < a.W; w += kWaves) {
        const size_t row = row0 + w;
        const bool ended = a.ended && a.ended[row];
        const double score = a.scores[row];
        const BeamPiece* p = a.pieces + row * a.splits;
        float top = -FLT_MAX;
        double sum = 0.0;
        if (!ended) {
            for (int i = lane; i < a.splits; i += kWave) top = fmaxf(top, p[i].top);
            top = wave_most(top);
            for (int i = lane; i < a.splits; i += kWave) sum += p[i].sum * exp(static_cast<double>(p[i].top) - top);
            sum = wave_sum(sum);
        }
        // rows with an infinity or NaN have no sum, and rows of -inf only a sum of zero
        const bool live = ended || (sum > 0.0 && sum < INFINITY && top < INFINITY);
        if (lane == 0) {
            shift[w] = live && fabs(score) < INFINITY ? (ended ? score : score - log(sum)) : -INFINITY;
            largest[w] = top;
        }
    }
    if (tid == 0) total = waiting = 0;
    __syncthreads();
    auto beam_of = [&](int list) { return static_cast<int>(static_cast<unsigned>(list) / static_cast<unsigned>(a.splits)); };
    auto place_of = [](int w, int token) { return static_cast<unsigned long long>(w) << 32 | static_cast<uint32_t>(token); };
    auto ended = [&](int w) { return a.ended && a.ended[row0 + w]; };
    // (the lists of a beam that has ended or has no candidates hold anything)
    auto score_of = [&](int list, const BeamEntry& e) -> double {
        const int w = beam_of(list);
        return shift[w] == -INFINITY || ended(w) || e.token < 0 ? -INFINITY : (static_cast<double>(e.logit) - largest[w]) + shift[w];
    };
    auto candidate = [&](int list, int depth) -> BeamCandidate {
        const BeamEntry e = entries[static_cast<size_t>(list) * a.count + depth];
        return {score_of(list, e), place_of(beam_of(list), e.token)};
    };
    auto own = [&](int w) -> BeamCandidate {                         // of a beam that has ended
        return ended(w) ? BeamCandidate{shift[w], place_of(w, a.end_token)} : BeamCandidate{-INFINITY, ~0ull};
    };
    // The bound: from each list's first entries, as many as there are threads for, neighbours in different groups.
    const int list0 = tid / deep, depth0 = tid - list0 * deep;
    const bool has = tid < lists * deep;
    const double score0 = has ? score_of(list0, mine) : -INFINITY;
    double best = score0;
    for (int list = tid + kMergeThreads; list < lists; list += kMergeThreads)     // (deep is 1)
        best = fmax(best, score_of(list, entries[static_cast<size_t>(list) * a.count]));
    groups.part[wave][lane] = best;
    const double nth = groups.nth(a.count - 1);
    if (tid == 0) bound_of = fmax(nth, -DBL_MAX);
    __syncthreads();
    double bound = bound_of;
    auto gather = [&](const BeamCandidate& c) {
        const int at = atomicAdd(&total, 1);
        if (at < kBeamRoom) found[at] = c;
    };
    // What reaches the bound of those entries, and the rest of the lists (few) whose last one of them does: all their entries at once. (Entry by
    // entry, one list's 16 took 9 us.)
    auto collect = [&](auto reaches) {
        auto rest = [&](int list) {
            if (deep == a.count) return;
            const int at = atomicAdd(&waiting, 1);
            if (at < kBeamRoom) {
                queue[at] = list;
                return;
            }
            for (int depth = deep; depth < a.count; depth++) {
                const BeamCandidate c = candidate(list, depth);
                if (!reaches(c.score)) break;
                gather(c);
            }
        };
        if (reaches(score0)) {
            gather({score0, place_of(beam_of(list0), mine.token)});
            if (depth0 == deep - 1) rest(list0);
        }
        for (int list = tid + kMergeThreads; list < lists; list += kMergeThreads) {
            const BeamCandidate c = candidate(list, 0);
            if (!reaches(c.score)) continue;
            gather(c);
            rest(list);
        }
        __syncthreads();
        const int left = a.count - deep, queued = min(waiting, kBeamRoom) * left;
        for (int i = tid; i < queued; i += kMergeThreads) {
            const int q = i / left;
            const BeamCandidate c = candidate(queue[q], deep + i - q * left);
            if (reaches(c.score)) gather(c);
        }
        if (a.ended)
            for (int w = tid; w < a.W; w += kMergeThreads) {
                const BeamCandidate c = own(w);
                if (reaches(c.score)) gather(c);
            }
        __syncthreads();
    };
    // A better bound from what was found, if it is one.
    auto better = [&]() {
        best = -INFINITY;
        for (int i = tid; i < min(total, kBeamRoom); i += kMergeThreads) best = fmax(best, found[i].score);
        groups.part[wave][lane] = best;
        const double nth = groups.nth(a.count - 1);
        if (tid == 0) {
            bound_of = fmax(nth, bound);
            total = waiting = 0;
        }
        __syncthreads();
        const bool risen = bound_of > bound;
        bound = bound_of;
        return risen;
    };
    const size_t out = static_cast<size_t>(blockIdx.x) * a.count;
    auto put = [&](int place, const BeamCandidate& c) {
        const bool some = c.score > -INFINITY;
        a.out_scores[out + place] = some ? static_cast<float>(c.score) : -INFINITY;
        a.out_beams[out + place] = some ? static_cast<int>(c.place >> 32) : -1;
        a.out_tokens[out + place] = some ? static_cast<int>(c.place & 0xFFFFFFFFu) : -1;
    };
    const BeamCandidate none = {-INFINITY, ~0ull};
    auto rank = [&](int got) {
        for (int i = tid; i < got; i += kMergeThreads) {
            const BeamCandidate c = found[i];
            int place = 0;
#pragma unroll 4
            for (int j = 0; j < got; j++) place += beam_before(found[j], c);
            if (place < a.count) put(place, c);
        }
    };
    // (Ends: a bound that has risen leaves out what had the one before, a candidate's score from the first time on. Some five rounds for 64 thousand.)
    for (;;) {
        collect([&](double x) { return x >= bound; });
        int got = total;
        if (got <= kBeamFew) {
            rank(got);
            for (int i = got + tid; i < a.count; i += kMergeThreads) put(i, none);
            return;
        }
        if (better()) continue;
        // Many equal ones: those above the bound, then the first that equal it, in the order of beams, pieces and lists.
        collect([&](double x) { return x > bound; });
        got = total;
        if (got > kBeamRoom) {                                       // (all of them are above it)
            better();
            continue;
        }
        rank(got);
        const int all = lists * a.count;
        for (int i0 = 0, turn = 0; i0 < all && got < a.count; i0 += kMergeThreads, turn ^= 1) {
            const int i = i0 + tid, list = static_cast<unsigned>(i) / static_cast<unsigned>(a.count), w = beam_of(list);
            BeamCandidate c = none;
            if (i < all) {
                if (!ended(w)) c = candidate(list, i - list * a.count);
                else if (i == w * a.splits * a.count) c = own(w);
            }
            const unsigned long long equal = __ballot(c.score == bound);
            if (lane == 0) part_count[turn][wave] = __popcll(equal);
            __syncthreads();
            int place = got + __popcll(equal & ((1ull << lane) - 1ull));
            for (int v = 0; v < kWaves; v++) {
                place += v < wave ? part_count[turn][v] : 0;
                got += part_count[turn][v];
            }
            if (c.score == bound && place < a.count) put(place, c);
        }
        for (int i = got + tid; i < a.count; i += kMergeThreads) put(i, none);
        return;
    }
}

// Vectors of a thread: a piece of 8192 logits, or one vector while that leaves CUs without work.
template <class L>
int beam_vectors(int B, int W, int V) {
    return static_cast<long long>(B) * W * divup(V, kBeamThreads * L::kMany * L::kPer) >= 2 * default_cu_count() ? L::kMany : 1;
}
template <class L>
int beam_splits(int B, int W, int V) { return divup(V, kBeamThreads * beam_vectors<L>(B, W, V) * L::kPer); }
inline bool beam_shape_ok(int B, int W, int V, int count) {
    return B > 0 && W > 0 && W <= kBeamWidth && V > 0 && count > 0 && count <= kBeamCount && B <= grid_limit(kMergeThreads) &&
           static_cast<long long>(B) * W * std::max(beam_splits<Logits16<Fp16>>(B, W, V), beam_splits<Logits32>(B, W, V)) <= grid_limit(kBeamThreads) &&
           static_cast<long long>(W) * (divup(V, kBeamThreads * 4) * static_cast<long long>(count) + 1) <= INT_MAX - kMergeThreads;
}
inline size_t beam_bytes(int B, int W, int count, int splits) {
    return static_cast<size_t>(B) * W * splits * (sizeof(BeamPiece) + count * sizeof(BeamEntry));
}

template <class L>
int launch_beams(BeamArgs a, void* workspace, size_t bytes, hipStream_t s) {
    a.splits = beam_splits<L>(a.B, a.W, a.V);
    if (bytes < beam_bytes(a.B, a.W, a.count, a.splits)) return FORGE_EINVAL;
    a.pieces = static_cast<BeamPiece*>(workspace);
    a.entries = reinterpret_cast<BeamEntry*>(a.pieces + static_cast<size_t>(a.B) * a.W * a.splits);
    const unsigned grid = static_cast<unsigned>(a.B) * a.W * a.splits;
    if (beam_vectors<L>(a.B, a.W, a.V) == L::kMany) beam_piece_kernel<L, L::kMany><<<grid, kBeamThreads, 0, s>>>(a);
    else beam_piece_kernel<L, 1><<<grid, kBeamThreads, 0, s>>>(a);
    const int st = launch_status();
    if (st != FORGE_OK) return st;
    beam_merge_kernel<<<static_cast<unsigned>(a.B), kMergeThreads, 0, s>>>(a);
    return launch_status();
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_beam_select_workspace_size(int B, int W, int V, int count) {
    if (!beam_shape_ok(B, W, V, count)) return 0;
    // of any type
    return beam_bytes(B, W, count, std::max(beam_splits<Logits16<Fp16>>(B, W, V), beam_splits<Logits32>(B, W, V)));
}

extern "C" int forge_beam_select(const void* logits, const float* scores, const uint8_t* ended, int end_token, float* out_scores,
                                 int32_t* out_beams, int32_t* out_tokens, int B, int W, int V, int count,
                                 long long batch_stride, long long beam_stride, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream)
{
    if (B <= 0 || W <= 0 || V <= 0 || count <= 0) return FORGE_OK;
    if (!beam_shape_ok(B, W, V, count) || !logits || !scores || !out_scores || !out_beams || !out_tokens || batch_stride < 0 ||
        beam_stride < 0 || (dtype != FORGE_FP16 && dtype != FORGE_BF16 && dtype != FORGE_FP32) ||
        (ended && (end_token < 0 || end_token >= V)) || !aligned(logits, dtype == FORGE_FP32 ? 4 : 2) || !workspace || !aligned(workspace, 16))
        return FORGE_EINVAL;
    const BeamArgs a{logits, scores, ended, out_scores, out_beams, out_tokens, nullptr, nullptr, batch_stride, beam_stride,
                     B, W, V, count, end_token, 0};
    hipStream_t s = as_stream(stream);
    if (dtype == FORGE_FP32) return launch_beams<Logits32>(a, workspace, workspace_bytes, s);
    return dtype == FORGE_FP16 ? launch_beams<Logits16<Fp16>>(a, workspace, workspace_bytes, s)
                               : launch_beams<Logits16<Bf16>>(a, workspace, workspace_bytes, s);
}
