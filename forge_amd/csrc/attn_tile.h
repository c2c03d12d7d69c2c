// One wave's attention over a tile of keys that lies in LDS, for FP16 and BF16.
//
// The wave owns 32 query rows. It multiplies S^T = K Q^T on
// 32 x 32 x 16 products: keys are the A operand's rows, queries the B operand's columns, and a lane
// ends up with 16 of a block's 32 scores of ONE query (lane l: query l % 32; register e: key 8 (e / 4) +
// 4 (l / 32) + e % 4). Row maxima and sums are then mostly inside a lane (one exchange with lane l ^ 32),
// and the probabilities, rounded in pairs, are as they stand the B operand of O^T = V^T P^T: a
// product's sum over keys may take them in any order, if V^T's operand takes the same one. That operand
// is 4 + 4 keys of one column of V, which the transposing LDS read gathers from V's rows.
// The running maximum m, sum l and O follow the published recurrence (online softmax), FP32; P is rounded to 16 bits for
// its product, which the matrix instructions take, and l sums the rounded weights, so that they add up to one (a prompt's errors in the 2-norm 2.6e-4
// of the result in FP16 and 2.0e-3 in BF16, against 2.0e-4 and 1.6e-3 with FP32 weights: the result's own rounding is
// most of both). O is rescaled only when some row's maximum has grown by more than 2^8 since the last time: until then P stays
// below 2^8, well inside both types.
//
// K and V tiles are rows of DP values (D padded with zeros) in 16-byte chunks, permuted in each row so that what
// LDS serves in one clock falls on different banks: one chunk of 16 rows of K, four chunks of 4 rows of V.
#pragma once

#include "float16_types.h"
#include "lds_dma.h"

#include <cfloat>

namespace forge_amd {

constexpr float kNoScore = -FLT_MAX;   // running maximum of a row that has seen nothing: no score is below it
constexpr float kRescale = 8.0f;
constexpr float kFar = 1048576.0f;

typedef short v4s __attribute__((ext_vector_type(4)));

// Four values of one column from four rows: each lane of 16 passes the address of 4 values of row
// (lane / 4), columns 4 (lane % 4) on; lane i receives column i of the four rows.
__device__ __forceinline__ v2u lds_read_tr(const int8_t* p) {
    return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) v4s*)p));
}

// The value of lane l ^ 32 combined with this lane's.
__device__ __forceinline__ float half_max(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Tile rows of DP values; physical chunk = logical chunk ^ swz(row).
template <int DP>
struct KvRows {
    static_assert(DP == 64 || DP == 96 || DP == 128 || DP == 256, "row lengths with a permutation");
    static constexpr int kChunks = DP / 8, kBytes = DP * 2;
    static __device__ __forceinline__ int swz_k(int r) {
        return DP == 64 ? (r >> 1) & 7 : DP == 96 ? (r >> 2) & 3 : r & 15;
    }
    static __device__ __forceinline__ int swz_v(int r) {
        return DP == 64 ? 4 * ((r >> 1) & 1) : DP == 96 ? 0 : 4 * (r & 3);
    }
};

// Two 16-bit values, those that are no finite numbers as zeros.
template <class T>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
    const uint32_t lo = (w & T::kInfinity) == T::kInfinity ? 0u : 0x0000FFFFu;
    const uint32_t hi = (w >> 16 & T::kInfinity) == T::kInfinity ? 0u : 0xFFFF0000u;
    return w & (lo | hi);
}

// Bits 0 to last.
__device__ __forceinline__ uint32_t bits_to(int last) {
    return last >= 31 ? ~0u : last < 0 ? 0u : (2u << last) - 1u;
}

template <class T, int DP, int KB>
struct AttnWave {
    using Rows = KvRows<DP>;
    static constexpr int kSteps = DP / 16, kOut = DP / 32;
    v4u q[kSteps];
    v16f o[kOut];
    float m, l;              // of query lane % 32; l: this lane's keys only
    float limit;             // a larger score has the weights taken again
    float low, shift;        // all weights are 2^-low of themselves; -(m + low)
    int lane, k_at, v_at;    // byte addresses in a tile, before the chunk permutation
    int k_x, v_x;            // the permutations, as byte masks

    __device__ __forceinline__ void init() {
        lane = threadIdx.x & (kWave - 1);
        const int half = lane >> 5, r = lane & 31, i = lane & 15, vr = 4 * half + i / 4;
        k_at = r * Rows::kBytes;
        k_x = (half ^ Rows::swz_k(r)) * 16;
        v_at = vr * Rows::kBytes + (i & 1) * 8;
        v_x = ((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ Rows::swz_v(vr)) * 16;
        m = kNoScore;
        limit = kNoScore;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < kOut; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[j][e] = 0.0f;
    }

    // The keys of the sequence. BF16 values may be as large as FP32 holds, and a sum of them must not pass that: the weights, each
    // up to 2^kRescale, are taken so low that all of them add up to less than one. BF16 has the range for it; FP16 has not,
    // and its values do not need it.
    __device__ __forceinline__ void keys(int n) { low = T::kWide ? kRescale + 33 - __builtin_clz(n) : 0.0f; }

    // D values of the query row at p, or zeros.
    __device__ __forceinline__ void load_q(const uint16_t* p, bool live, int D) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            const int d = 16 * s + 8 * (lane >> 5);
            q[s] = live && d < D ? *reinterpret_cast<const v4u*>(p + d) : v4u{0u, 0u, 0u, 0u};
        }
    }

    // The order of a block's N products and the LDS reads of their operands, R each: those of the first
    // `ahead` products, then one product and the reads of the one `ahead` further on. Left to itself the compiler
    // reads one or two ahead and each product waits for LDS.
    static constexpr int kAhead = 6;
    template <int N, int R, int AHEAD>
    static __device__ __forceinline__ void interleave() {
        __builtin_amdgcn_sched_group_barrier(0x100, R * (AHEAD < N ? AHEAD : N), 0);
#pragma unroll
        for (int i = 0; i < N; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
        }
    }

    using Scores = v16f[KB];
    using Weights = v4u[KB][2];

    // Scores of a tile of 32 KB keys; products in a row go to different sums.
    __device__ __forceinline__ void scores(const int8_t* ks, Scores& s) const {
#pragma unroll
        for (int st = 0; st < kSteps; st++)
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                const v4u k = *reinterpret_cast<const v4u*>(ks + 32 * kb * Rows::kBytes + k_at + ((32 * st) ^ k_x));
                const v16f zero = {};
                s[kb] = T::mfma32(k, q[st], st == 0 ? zero : s[kb]);
            }
        interleave<KB * kSteps, 1, kAhead>();
    }

    // seen(kb) has a bit for each key of block kb that this lane's row sees.
    template <class Seen>
    __device__ __forceinline__ void mask(Scores& s, const Seen& seen) const {
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            const uint32_t bits = seen(kb) >> (4 * (lane >> 5));
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (!(bits & (1u << (8 * (e / 4) + e % 4)))) s[kb][e] = -INFINITY;
        }
    }

    // The row's largest score, in the exponent's units.
    __device__ __forceinline__ float largest(const Scores& s, float scale2) const {
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {                                // four chains of maxima of three
            mx[c] = s[0][4 * c];
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[c] = fmaxf(mx[c], s[kb][4 * c + e]);
        }
        return half_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))) * scale2;
    }

    // The weights 2^(unit s + shift); returns their sum.
    __device__ __forceinline__ float weights(const Scores& s, float unit, float shift, Weights& p) const {
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * h + 2 * d], unit, shift));
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * h + 2 * d + 1], unit, shift));
                    p[kb][h][d] = T::pack(x, y);
                    sum[h] = T::add_pair(p[kb][h][d], sum[h]);
                }
        return sum[0] + sum[1];
    }

    // The maximum takes x in. Rows whose scores lie far from zero have their weights always taken again: a fused multiply-add does
    // not round scale2 s, as the maximum was, and that difference (2^-4 of an exponent at kFar) would at last move
    // all weights of a row out of their type.
    __device__ __forceinline__ void raise(float x) {
        m = fmaxf(m, x);
        limit = fabsf(m) > kFar && m != kNoScore ? -INFINITY : m + kRescale;
        shift = -(m + low);
    }

    // The exponents in place of the scores, each product rounded as the maximum's was.
    __device__ __forceinline__ void exponents(Scores& s, float scale2) const {
#pragma clang fp contract(off)
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = s[kb][e] * scale2;
                s[kb][e] = x - m;
            }
    }

    // O += P V of a tile.
    __device__ __forceinline__ void values(const int8_t* vs, const Weights& p) {
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < kOut; j++) {
                    const int8_t* at = vs + (32 * kb + 16 * h) * Rows::kBytes + v_at + ((64 * j) ^ v_x);
                    const v2u lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * Rows::kBytes);
                    const v4u v = {lo[0], lo[1], hi[0], hi[1]};
                    o[j] = T::mfma32(v, p[kb][h], o[j]);
                }
        interleave<2 * KB * kOut, 2, kAhead>();
    }

    // A tile of V (32 KB KS rows at v, one wave's at vs) that some rows of the workgroup see in part, before its products: these would
    // take a value times the zero weight of a row that does not see it, which is NaN where that value is infinite or
    // NaN. Such values are added to the sums of the rows that see them (their weights are positive) and are zeros then. All waves
    // call it, between the barrier that makes the tile whole and the products; `odd`, in LDS, holds no number of this tile yet.
    // us of a prompt of 9001, 32 / 8 heads of 128, and of one of 1024, 8 heads: finite values 709 and 17.4, a NaN in the first
    // 703 and 17.4, infinities in one of a hundred values 1161 and 78, NaN only 1296 and 92.
    template <int W, int KS, class Seen>
    __device__ __forceinline__ void take_odd_values(int8_t* v, const int8_t* vs, int wave, int number, int* odd, const Seen& seen) {
        constexpr int kShare = 32 * KB * KS * Rows::kBytes / W;      // each wave looks through a part
        static_assert(kShare % 1024 == 0, "whole instructions");
        v4u* at = reinterpret_cast<v4u*>(v + wave * kShare + 16 * lane);
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < kShare / 1024; i++) {
            const v4u x = at[kWave * i];
#pragma unroll
            for (int d = 0; d < 4; d++) z = T::times_zero(x[d], z);
        }
        if (z != 0.0f) *odd = number;
        wait_lgkm0();
        lds_barrier();
        if (__builtin_amdgcn_readfirstlane(*odd) != number) return;
        add_odd_values(vs, seen);
        wait_lgkm0();
        lds_barrier();
#pragma unroll 1
        for (int i = 0; i < kShare / 1024; i++) {
            const v4u x = at[kWave * i];
            at[kWave * i] = v4u{finite_or_zero<T>(x[0]), finite_or_zero<T>(x[1]), finite_or_zero<T>(x[2]), finite_or_zero<T>(x[3])};
        }
        wait_lgkm0();
        lds_barrier();
    }
    template <class Seen>
    __device__ __forceinline__ void add_odd_values(const int8_t* vs, const Seen& seen) {
#pragma unroll 1
        for (int k = 0; k < 32 * KB; k++) {
            const int8_t* row = vs + k * Rows::kBytes;
            float z = 0.0f;
            if (lane < Rows::kChunks) {
                const v4u x = *reinterpret_cast<const v4u*>(row + 16 * lane);
#pragma unroll
                for (int d = 0; d < 4; d++) z = T::times_zero(x[d], z);
            }
            if (!__any(z != 0.0f)) continue;
            const bool on = seen(k >> 5) >> (k & 31) & 1u;
#pragma unroll
            for (int j = 0; j < kOut; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const v2u x = *reinterpret_cast<const v2u*>(row + ((4 * j + c) ^ Rows::swz_v(k)) * 16 + 8 * (lane >> 5));
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float y = T::widen(static_cast<uint16_t>(x[e / 2] >> (16 * (e & 1))));
                        o[j][4 * c + e] += on && !(fabsf(y) < INFINITY) ? y : 0.0f;
                    }
                }
        }
    }

    // A tile from its scores on; masked if `masked`. `first`: nothing has been summed yet. (Both uniform.)
    template <class Seen>
    __device__ __forceinline__ void finish(Scores& s, const int8_t* vs, float scale2, bool first, bool masked, const Seen& seen) {
        if (masked) mask(s, seen);
        if (first) raise(largest(s, scale2));
        Weights p;
        float sum = weights(s, scale2, shift, p);
        const float mx = largest(s, scale2);
        // A maximum that has grown is met seldom: the weights are taken again. (The compiler takes the ones above where nothing has
        // grown, so that they wait for the maximum after all.)
        if (__any(mx > limit)) {
            const float was = m;
            raise(mx);
            const float f = __builtin_amdgcn_exp2f(was - m);
            l *= f;
#pragma unroll
            for (int j = 0; j < kOut; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[j][e] *= f;
            exponents(s, scale2);
            sum = weights(s, 1.0f, -low, p);
        }
        l += sum;
        values(vs, p);
    }

    // Joining KS waves (wave, wave + 1, .. from a multiple of KS on) that have the same rows and other keys, in
    // wave order: each leaves its state in LDS, and after a barrier wave ks takes every KS-th block of 32
    // columns from ks on. put(j, e, sums of columns 32 j + 8 e + 4 (lane / 32) .. + 3, maximum, sum of the weights).
    template <int W>
    struct Shared {
        v4f sums[W][kOut * 4][kWave];
        v2f stat[W][32];
    };
    template <int W>
    __device__ __forceinline__ void leave(Shared<W>* sh, int wave, bool live) const {
        const float sum = half_sum(l);
        if (lane < 32) sh->stat[wave][lane] = v2f{m, sum};
        if (!live) return;                                           // a row that nobody asks for
#pragma unroll
        for (int j = 0; j < kOut; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                sh->sums[wave][4 * j + e][lane] = v4f{o[j][4 * e], o[j][4 * e + 1], o[j][4 * e + 2], o[j][4 * e + 3]};
    }
    template <int KS, int W, class Put>
    __device__ __forceinline__ void join(const Shared<W>* sh, int wave, const Put& put) const {
        const int ks = wave % KS, w0 = wave - ks;
        float top = kNoScore, sum = 0.0f, f[KS];
#pragma unroll
        for (int v = 0; v < KS; v++) {
            f[v] = sh->stat[w0 + v][lane & 31][0];
            top = fmaxf(top, f[v]);
        }
#pragma unroll
        for (int v = 0; v < KS; v++) {
            f[v] = __builtin_amdgcn_exp2f(f[v] - top);
            sum = __builtin_fmaf(f[v], sh->stat[w0 + v][lane & 31][1], sum);
        }
#pragma unroll
        for (int j = 0; j < kOut; j++) {
            if (j % KS != ks) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int v = 0; v < KS; v++) {
                    const v4f y = sh->sums[w0 + v][4 * j + e][lane];
#pragma unroll
                    for (int c = 0; c < 4; c++) s[c] = __builtin_fmaf(f[v], y[c], s[c]);
                }
                put(j, e, s, top, sum);
            }
        }
    }
};

}  // namespace forge_amd
