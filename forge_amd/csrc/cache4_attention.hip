// Attention of a few new tokens per sequence over the 4-bit paged cache (cache4.h): one token or a tree of up to 64 drafts,
// as cache_attention.
//
// With k = m + s n the score of row r and key j is scale (s_j (q_r . n_j) + m_j sum q_r), and the result is
// (sum_j p_rj v_j) / sum_j p_rj with v_j = m'_j + s'_j n'_j, so the products are of 16-bit numbers with the integers themselves, which FP16 holds
// exactly, and steps and lowest values enter in FP32: no key or value is rounded to 16 bits, and what a row does not see (its
// integers are always finite) is left out by a select of its weight.
//
// A wave owns 16 RT rows and takes blocks of 16 keys, two at a time, on 16 x 16 x 32 products, S^T = K Q^T and O^T = V^T P^T as in attn_tile.h. All of
// its operands come straight from memory: a lane's 8 values of one key are a word, and its word of four keys lies together (cache4.h).
// Nibbles are FP16 subnormals n 2^-20, at bits 4 and 20 of a register; the power of two goes into the scores and the result, and queries
// are scaled by one of their own per row (BF16 queries fit FP16 then). The matrix unit aligns the 8 products of a lane by the exponents of
// their factors, that of a subnormal being 2^-14, and drops what lies 24 bits below: 2^-18 of the largest query, or weight, of the 8.
// Masked where they are, at bits 0 and 16 too (n 2^-24, of which 2^-14 is dropped), they take one shift for 8 values instead of
// three, 4 % of the time of 6 trees (below).
// Weights w = p s' are rounded to FP16, in either type, the row's largest at 2^4 or above (as far as a factor of 2^127 brings it there, which for
// p of 2^-low is up to steps of 2^(low - 123); BF16's smaller ones lose bits); sums are FP32. v is taken as (m' + 8 s') + s' (n' - 8):
// sum w n' less 8 times the sum of the same rounded w, so that a rounding weighs with n' - 8 (a result's error in the 2-norm, FP16 values: 2.4e-4 to
// 2.8e-4; with n' 5.4e-4; rounding the exact result alone 2.1e-4).
//
// Bound: reading the cache for up to 16 rows: one token over 16 sequences of 278 thousand keys, 32 / 8 heads of 128, 55 us, 5.5 TB/s of 303 MB (and
// 4.7 for the join of the chunks; 16-bit caches read 3.8 times as much). Many rows: the vector units. 6 trees of 16 drafts, 32 / 4 heads of
// 128, over 119 thousand keys take 70 us (445 TFLOP/s): 410 vector and 32 matrix instructions for 32 rows and 32 keys, of them 120 for the operands, 40 for
// steps and lowest values and 13 (16 with the exponential's rate) per score. Sharing the operands of four waves in LDS took 16 % of the
// instructions away and 11 % more time: the waves wait for each other at every tile.
#include "cache4.h"
#include "cache_split.h"

#include <type_traits>

namespace forge_amd {

struct Cache4Args : CacheArgs {
    const uint8_t* cache;
    int2* info;          // by sequence: its first slot and its chunks
    int slots, target, least, grain, fit;   // find_chunk; slots 0: chunks of `chunk` keys, `chunks` of them for each sequence
};

// Chunks by what the sequences hold: a length, in whole `grain` keys and of `least` at least, that makes `target` of all keys together;
// with `fit` (64 sequences at most) up to a quarter more, while the sequences' last ones make them more than `target`. Each sequence then has its
// chunks of equal length. A grid row takes a chunk; target + B of them are always enough, and go to the sequences in order (one may be left
// empty by the rounding). All of it follows from the lengths, which every wave looks through.
struct Cache4Chunk {
    int b, index, length;        // sequence, chunk of it, keys of its chunks
    int first;                   // of them
};
// Sum over the lanes up to this one.
__device__ __forceinline__ int lanes_before(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}
__device__ __forceinline__ bool find_chunk(const Cache4Args& a, int slot, int lane, Cache4Chunk* c) {
    auto keys_of = [&](int b) { return b < a.B ? cache_keys(a, b) : 0; };
    const int mine = keys_of(lane);
    int keys = mine;
    for (int b = kWave; b < a.B; b += kWave) keys += keys_of(b + lane);
    const int total = __builtin_amdgcn_readlane(lanes_before(keys), 63);   // (2^30 at most: the launcher's check)
    auto grains = [&](unsigned keys) { return static_cast<int>((keys + a.grain - 1u) & -a.grain); };
    auto share = [&](unsigned keys) { return (keys + a.target - 1u) / static_cast<unsigned>(a.target); };   // of `target` chunks
    auto chunks_of = [&](int k) { return static_cast<int>((static_cast<unsigned>(k) + c->length - 1u) / static_cast<unsigned>(c->length)); };
    c->length = __builtin_amdgcn_readfirstlane(max(grains(share(total)), a.least));
    if (a.fit) {
        const int most = c->length + c->length / 4;
        for (int i = 0; i < 3; i++) {
            const int all = __builtin_amdgcn_readlane(lanes_before(chunks_of(mine)), 63);
            if (all <= a.target) break;
            c->length = __builtin_amdgcn_readfirstlane(grains(min(share(static_cast<unsigned>(c->length) * all), static_cast<unsigned>(most))));
        }
    }
    int base = 0;
    for (int b = 0; b < a.B; b += kWave) {
        const int n = chunks_of(b == 0 ? mine : keys_of(b + lane));
        const int upto = base + lanes_before(n);
        const unsigned long long past = __ballot(upto > slot);
        if (past) {
            const int l = __builtin_ctzll(past);
            const unsigned k = cache_keys(a, b + l), mine_n = __builtin_amdgcn_readlane(n, l);
            c->b = b + l;
            c->first = __builtin_amdgcn_readlane(upto, l) - mine_n;
            c->index = slot - c->first;
            c->length = grains((k + mine_n - 1u) / mine_n);
            return true;
        }
        base = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Values 2 i and 2 i + 1 of a word as half pairs, n 2^-20 each.
constexpr uint32_t kNibble = 0x00F000F0u;
__device__ __forceinline__ v4u nibble_pairs(uint32_t w) {
    return v4u{(w << 4) & kNibble, w & kNibble, (w >> 4) & kNibble, (w >> 8) & kNibble};
}

__device__ __forceinline__ float swap16_max(float x) {
    const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap16_sum(float x) {
    const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Over the four lanes of a column.
__device__ __forceinline__ float column_max(float x) { return half_max(swap16_max(x)); }
__device__ __forceinline__ float column_sum(float x) { return half_sum(swap16_sum(x)); }

template <int U>
struct Words4 {
    // Operands of 16 words for all 8 values of each (full sets), of 8 words for the first and second half of the lanes (a half set).
    static constexpr int kFull = U == 2 ? 0 : U == 8 ? 2 : 1, kHalf = U == 2 || U == 6, kSets = kFull + kHalf;
    static constexpr int kOut = 8 * kFull + 4 * kHalf;   // products of 16 columns of the result
    static constexpr int kRow = 32 * U + 4;              // floats of a row in LDS
    static __device__ __forceinline__ int word(int s, int n) {
        return s < kFull ? min(16 * s + n, 4 * U - 1) : 16 * kFull + (n & 7);
    }
};

template <int U>
struct Block4 {   // a lane's part of 16 keys
    uint32_t k[U];
    v4u v[Words4<U>::kSets];
    v4u num[2];           // numbers of keys 4 g to 4 g + 3
};

constexpr int kMostE = 127;   // of a factor 2^e that FP32 holds

// One row tile's softmax state (the lane's column).
template <int U>
struct Rows4 {
    v4u q[U];
    v4f o[Words4<U>::kOut];
    float unit, qsum;        // of a score; the sum of the row's queries, in exponents
    float shift, limit;      // exponents are scores + shift; above limit the shift is lowered (-FLT_MAX: none yet)
    float l, c, u;           // this lane's sums of p, of p (m' + 8 s') and of the rounded weights
    float f, top;            // weights are f p s'; the largest p s' when f was chosen
    int e;                   // f = 2^e
    __device__ __forceinline__ void scale(float by) {
#pragma unroll
        for (int j = 0; j < Words4<U>::kOut; j++) o[j] *= by;
        u *= by;
    }
};

__device__ const uint4 kNoNumbers[8] = {};   // those of a page that is not there

// Waves of a SIMD that the registers are to leave room for.
constexpr int cache4_waves(int U, int RT) { return U <= 4 ? (RT == 1 ? 3 : 2) : RT == 1 ? 2 : 1; }

template <class T, int U, int RT, int RS, int KS>
__global__ __launch_bounds__(64 * RS * KS, cache4_waves(U, RT)) void cache4_attention_kernel(Cache4Args a)
{
#pragma clang fp contract(off)
    using Words = Words4<U>;
    constexpr int W = RS * KS, kRowTiles = RT * RS;
    extern __shared__ __align__(1024) int8_t lds[];
    float* sums = reinterpret_cast<float*>(lds);                     // W x 16 x kRow, one row tile of each wave at a time
    v2f* stat = reinterpret_cast<v2f*>(sums + W * 16 * Words::kRow);  // W x 16
    int* page_of = reinterpret_cast<int*>(stat + W * 16);

    const int group = a.group, rows = a.T * group;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x & (kWave - 1), col = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x;
    int b, chunk = blockIdx.y, set, chunk_keys;
    if (a.slots) {
        Cache4Chunk c;
        if (!find_chunk(a, blockIdx.y, lane, &c)) return;
        b = c.b;
        chunk = c.index;
        set = blockIdx.z;
        chunk_keys = c.length;
        if (hk == 0 && set == 0 && chunk == 0 && threadIdx.x == 0) a.info[b] = int2{c.first, (cache_keys(a, b) + chunk_keys - 1) / chunk_keys};
    } else {
        b = udiv_magic(blockIdx.z, a.mg_sets);
        set = blockIdx.z - b * a.sets;
        chunk_keys = a.chunk;
    }
    b = __builtin_amdgcn_readfirstlane(b);                           // (the same in all lanes, which the compiler does not see)
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    set = __builtin_amdgcn_readfirstlane(set);
    chunk_keys = __builtin_amdgcn_readfirstlane(chunk_keys);
    const int rs = wave / KS, ks = wave % KS;
    const int key0 = chunk * chunk_keys, page_mask = (1 << a.page_shift) - 1, page0 = key0 >> a.page_shift;
    const int last_page = min((key0 + chunk_keys - 1) >> a.page_shift, a.width - 1);
    for (int p = page0 + threadIdx.x; p <= last_page; p += 64 * W) {
        const int pg = a.table[static_cast<size_t>(b) * a.width + p];
        page_of[p - page0] = pg >= 0 && pg < a.pages ? pg : -1;
    }
    auto row_of = [&](auto* base, int r) {                           // of q and out
        const int t = udiv_magic(r, a.mg_group);
        return base + ((static_cast<size_t>(b) * a.T + t) * a.Hq + hk * group + (r - t * group)) * a.D;
    };
    const int row0 = (set * kRowTiles + rs * RT) * 16;               // this wave's rows

    Rows4<U> st[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int row = row0 + 16 * rt + col;
        const bool live = row < rows;
        v4u raw[U];
        const uint16_t* src = row_of(a.q, live ? row : 0);
#pragma unroll
        for (int c = 0; c < U; c++) {
            const int d = 8 * (g * U + c);
            raw[c] = live && d < a.D ? *reinterpret_cast<const v4u*>(src + d) : v4u{0u, 0u, 0u, 0u};
        }
        float x[U][8], most = 0.0f, odd = 0.0f;
#pragma unroll
        for (int c = 0; c < U; c++) {
            widen8<T>(raw[c], x[c]);
#pragma unroll
            for (int i = 0; i < 8; i++) most = fmaxf(most, fabsf(x[c][i]));
#pragma unroll
            for (int i = 0; i < 4; i++) odd = T::times_zero(raw[c][i], odd);
        }
        most = column_max(most);
        // the row's largest query becomes 2^14 to 2^15; rows that are not finite become NaN
        const int up = most > 0.0f && most < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
        float sum = odd;
#pragma unroll
        for (int c = 0; c < U; c++) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                y[i] = ldexpf(x[c][i], up);
                sum += y[i];
            }
            st[rt].q[c] = narrow8<Fp16>(y);
        }
        // (a unit past FP32 belongs to scores that only differ by more than any exponent)
        st[rt].unit = fminf(ldexpf(a.scale * 1.44269504f, 20 - up), 0x1p126f);
        st[rt].qsum = column_sum(sum) * 0x1p-20f * st[rt].unit;
        st[rt].shift = 0.0f;
        st[rt].limit = -FLT_MAX;
        st[rt].l = st[rt].c = st[rt].u = st[rt].top = 0.0f;
        st[rt].e = kMostE;
        st[rt].f = 0x1p127f;
#pragma unroll
        for (int j = 0; j < Words::kOut; j++) st[rt].o[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int keys = cache_keys(a, b), len = max(a.lens[b], 0), n = min(keys - key0, chunk_keys);
    if (n <= 0) return;
    // all weights are 2^-low of themselves, so that no sum of values passes FP32 (those of a head span twice BF16's range)
    const float low = kRescale + 35 - __builtin_clz(keys);
    __syncthreads();
    const int open = len - key0;                                     // keys of this chunk that every row sees

    const size_t piece = static_cast<size_t>(32 * U + 8) << a.page_shift;
    const uint32_t at_v = 16u * U << a.page_shift, at_num = 32u * U << a.page_shift;
    const uint32_t lane_k = 16 * U * col + 4 * U * g;
    struct Pages { int pg[2]; };
    auto look = [&](int tile) {                                      // the pages of a tile (past the last one: any)
        Pages p;
#pragma unroll
        for (int h = 0; h < 2; h++) p.pg[h] = page_of[((key0 + min(32 * tile + 16 * h, n - 1)) >> a.page_shift) - page0];
        return p;
    };
    auto load = [&](Block4<U> (&t)[2], int tile, const Pages& pages) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int pg = __builtin_amdgcn_readfirstlane(pages.pg[h]);
            const uint8_t* p = a.cache + (static_cast<size_t>(max(pg, 0)) * a.Hkv + hk) * piece;
            const uint32_t r = (key0 + 32 * tile + 16 * h) & page_mask;
            const uint8_t* pk = p + r * (16 * U) + lane_k;
            if constexpr (U % 4 == 0) {
#pragma unroll
                for (int c = 0; c < U; c += 4) *reinterpret_cast<v4u*>(t[h].k + c) = *reinterpret_cast<const v4u*>(pk + 4 * c);
            } else if constexpr (U % 2 == 0) {
#pragma unroll
                for (int c = 0; c < U; c += 2) *reinterpret_cast<v2u*>(t[h].k + c) = *reinterpret_cast<const v2u*>(pk + 4 * c);
            } else {
#pragma unroll
                for (int c = 0; c < U; c++) t[h].k[c] = *reinterpret_cast<const uint32_t*>(pk + 4 * c);
            }
#pragma unroll
            for (int s = 0; s < Words::kSets; s++)
                t[h].v[s] = *reinterpret_cast<const v4u*>(p + at_v + r * (16 * U) + 64 * U * g + 16 * Words::word(s, col));
            // (global addresses, or the choice makes flat loads, which LDS reads wait for)
            typedef __attribute__((address_space(1))) const v4u* Numbers;
            const Numbers pn = pg >= 0 ? (Numbers)(p + at_num + r * 8) : (Numbers)kNoNumbers;
            t[h].num[0] = pn[2 * g];
            t[h].num[1] = pn[2 * g + 1];
        }
    };

    // 32 keys from k0 on; masked: some rows do not see all of them.
    auto take = [&](const Block4<U> (&t)[2], int k0, auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        float vs[2][4], vm[2][4];
        v4f x[RT][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4f s[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) s[rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < U; c++) {
                const v4u k = nibble_pairs(t[h].k[c]);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) s[rt] = Fp16::mfma16(k, st[rt].q[c], s[rt]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t kn = t[h].num[e >> 1][2 * (e & 1)], vn = t[h].num[e >> 1][2 * (e & 1) + 1];
                const float step = T::widen(static_cast<uint16_t>(kn & 0xFFFFu)), least = T::widen(static_cast<uint16_t>(kn >> 16));
                vs[h][e] = T::widen(static_cast<uint16_t>(vn & 0xFFFFu));
                vm[h][e] = __builtin_fmaf(8.0f, vs[h][e], T::widen(static_cast<uint16_t>(vn >> 16)));
#pragma unroll
                for (int rt = 0; rt < RT; rt++)                      // (a BF16 key's step times s, up to 2^7, may pass FP32)
                    x[rt][h][e] = __builtin_fmaf(s[rt][e], step * st[rt].unit, __builtin_fmaf(least, st[rt].qsum, st[rt].shift));
            }
        }
        v4u weights[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            Rows4<U>& r = st[rt];
            uint32_t bits = ~0u;
            if constexpr (kMasked) {
                const int row = row0 + 16 * rt + col, token = udiv_magic(min(row, rows - 1), a.mg_group);
                const unsigned long long drafts =
                    a.tree ? static_cast<unsigned long long>(a.tree[static_cast<size_t>(b) * a.T + token]) : ~0ull >> (63 - token);
                const int d = open - k0;                             // bits below d: the cache; from d on: drafts
                bits = bits_to(d - 1);
                if (d < 32) bits |= d >= 0 ? static_cast<uint32_t>(drafts << d) : d > -64 ? static_cast<uint32_t>(drafts >> -d) : 0u;
                bits = (bits & bits_to(n - 1 - k0)) >> (4 * g);
            }
            auto on = [&](int h, int e) { return (bits >> (16 * h + e) & 1u) != 0u; };
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (kMasked && !on(h, e)) x[rt][h][e] = -INFINITY;
                    mx = fmaxf(mx, x[rt][h][e]);
                }
            if (__any(mx > r.limit)) {                               // a maximum that has grown
                const float most = column_max(mx);
                const bool grown = most > r.limit, none = r.limit == -FLT_MAX;
                const float to = grown ? r.shift - (most + low) : r.shift, d = to - r.shift;
                const float down = none ? 1.0f : __builtin_amdgcn_exp2f(d);
                // A shift far from zero is rounded by more than the exponents' own distances: those of this tile are taken relative to its
                // maximum itself then, or some would lie above every limit (from 2^32 on past FP32). `to` is at most the shift before.
                const bool far = grown && fabsf(to) > kFar;
                const float base = far ? most : 0.0f, rest = far ? -low : d;
                if (grown) r.limit = kRescale - low;
                r.shift = to;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[rt][h][e] = x[rt][h][e] - base + rest;
                r.l *= down;
                r.c *= down;
                r.top *= down;
                const int e = r.top > 0.0f ? max(-120, min(kMostE, 5 - __builtin_amdgcn_frexp_expf(r.top))) : kMostE;
                r.scale(ldexpf(down, e - r.e));
                r.e = e;
                r.f = ldexpf(1.0f, e);
            }
            float w[2][4], wx = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = __builtin_amdgcn_exp2f(x[rt][h][e]);
                    r.l += p;
                    r.c = __builtin_fmaf(p, kMasked && !on(h, e) ? 0.0f : vm[h][e], r.c);
                    w[h][e] = p * (kMasked && !on(h, e) ? 0.0f : vs[h][e]);
                    wx = fmaxf(wx, w[h][e]);
                }
            if (__any(wx * r.f > 32768.0f)) {                        // weights that FP16 would not hold
                r.top = fmaxf(r.top, column_max(wx));
                const int e = max(-120, min(r.e, 5 - __builtin_amdgcn_frexp_expf(r.top)));
                r.scale(ldexpf(1.0f, e - r.e));
                r.e = e;
                r.f = ldexpf(1.0f, e);
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                weights[rt][2 * h] = Fp16::pack(w[h][0] * r.f, w[h][1] * r.f);
                weights[rt][2 * h + 1] = Fp16::pack(w[h][2] * r.f, w[h][3] * r.f);
                r.u = Fp16::add_pair(weights[rt][2 * h], Fp16::add_pair(weights[rt][2 * h + 1], r.u));
            }
        }
#pragma unroll
        for (int s = 0; s < Words::kSets; s++) {
            constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;
            const bool full = s < Words::kFull;
#pragma unroll
            for (int half = 0; half < (full ? 2 : 1); half++) {
                const uint32_t sel = full ? (half ? kHigh : kLow) : (col < 8 ? kLow : kHigh);
                const v4u w = {__builtin_amdgcn_perm(t[0].v[s][1], t[0].v[s][0], sel), __builtin_amdgcn_perm(t[0].v[s][3], t[0].v[s][2], sel),
                         __builtin_amdgcn_perm(t[1].v[s][1], t[1].v[s][0], sel), __builtin_amdgcn_perm(t[1].v[s][3], t[1].v[s][2], sel)};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v4u v = (i == 0 ? w << 4 : w >> (4 * (i - 1))) & kNibble;
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        v4f& o = st[rt].o[8 * s + 4 * half + i];
                        o = Fp16::mfma16(v, weights[rt], o);
                    }
                }
            }
        }
    };

    // The wave's tiles, every KS-th, loaded one ahead and their pages looked up two ahead: those that all rows see whole, then the others.
    const int tiles = (n + 31) / 32, whole_tiles = max(min(open, n), 0) / 32;
    int tile = ks;
    Block4<U> t[2][2];
    Pages next = look(tile);
    load(t[0], tile, next);
    next = look(tile + KS);
    bool second = false;
    while (tile < whole_tiles) {
        load(t[1], tile + KS, next);
        next = look(tile + 2 * KS);
        take(t[0], 32 * tile, std::false_type{});
        tile += KS;
        second = tile >= whole_tiles;
        if (second) break;
        load(t[0], tile + KS, next);
        next = look(tile + 2 * KS);
        take(t[1], 32 * tile, std::false_type{});
        tile += KS;
    }
    if (second) {
#pragma unroll
        for (int h = 0; h < 2; h++) t[0][h] = t[1][h];
    }
    for (; tile < tiles; tile += KS) {
        load(t[1], tile + KS, next);
        next = look(tile + 2 * KS);
        take(t[0], 32 * tile, std::true_type{});
#pragma unroll
        for (int h = 0; h < 2; h++) t[0][h] = t[1][h];
    }

    // The KS waves of the same rows are joined in LDS, a row tile at a time.
    const bool whole = keys <= chunk_keys;                           // the only chunk: the result itself
    const size_t part0 = (a.slots ? static_cast<size_t>(hk) * a.slots + blockIdx.y : (static_cast<size_t>(b) * a.Hkv + hk) * a.chunks + chunk) * rows;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const Rows4<U>& r = st[rt];
        __syncthreads();                                             // the page list, the tile before
        const float l = column_sum(r.l), c = column_sum(r.c), u = 8.0f * column_sum(r.u);
        float* mine = sums + (wave * 16 + col) * Words::kRow;
        auto value = [&](int j, int e) { return ldexpf(r.o[j][e] * 0x1p20f - u, -r.e) + c; };
#pragma unroll
        for (int e = 0; e < 4; e++) {
#pragma unroll
            for (int s = 0; s < Words::kFull; s++) {
                const int w = 16 * s + 4 * g + e;                    // value 2 i + half of the word is product 4 half + i
                if (w >= 4 * U) continue;
                *reinterpret_cast<v4f*>(mine + 8 * w) = v4f{value(8 * s, e), value(8 * s + 4, e), value(8 * s + 1, e), value(8 * s + 5, e)};
                *reinterpret_cast<v4f*>(mine + 8 * w + 4) = v4f{value(8 * s + 2, e), value(8 * s + 6, e), value(8 * s + 3, e), value(8 * s + 7, e)};
            }
            if constexpr (Words::kHalf != 0) {
                const int at = 4 * g + e, w = 16 * Words::kFull + (at & 7);
#pragma unroll
                for (int i = 0; i < 4; i++) mine[8 * w + 2 * i + (at >> 3)] = value(8 * Words::kFull + i, e);
            }
        }
        if (g == 0) stat[wave * 16 + col] = v2f{r.limit == -FLT_MAX ? kNoScore : -(r.shift + low), l};
        __syncthreads();
        const int quads = a.D / 4;
        for (int i = threadIdx.x; i < RS * 16 * quads; i += 64 * W) {
            const int rr = i / quads, d = 4 * (i - rr * quads), set_row = rr >> 4, cc = rr & 15;
            const int row = (set * kRowTiles + set_row * RT + rt) * 16 + cc;
            if (row >= rows) continue;
            float top = kNoScore, sum = 0.0f;
#pragma unroll
            for (int v = 0; v < KS; v++) top = fmaxf(top, stat[(set_row * KS + v) * 16 + cc][0]);
            v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < KS; v++) {
                const v2f ml = stat[(set_row * KS + v) * 16 + cc];
                const float f = __builtin_amdgcn_exp2f(ml[0] - top);
                sum = __builtin_fmaf(f, ml[1], sum);
                const v4f z = *reinterpret_cast<const v4f*>(sums + ((set_row * KS + v) * 16 + cc) * Words::kRow + d);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(f, z[e], y[e]);
            }
            if (whole) {
                const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
                *reinterpret_cast<v2u*>(row_of(a.out, row) + d) = v2u{T::pack(y[0] * inv, y[1] * inv), T::pack(y[2] * inv, y[3] * inv)};
            } else {
                *reinterpret_cast<v4f*>(a.part + (part0 + row) * a.D + d) = y;
                if (d == 0) *reinterpret_cast<v2f*>(a.stat + (part0 + row) * 2) = v2f{top, sum};
            }
        }
    }
}

// W waves join the chunks of one row: their parts of LPR lanes of 4 values take every kSets-th chunk, four in flight, with the running
// maximum of a softmax; the parts are joined in a fixed order.
template <class T, int LPR, int W>
__global__ __launch_bounds__(256) void cache4_join_kernel(Cache4Args a)
{
    static_assert(W == 1 || W == 4, "a wave's row, or a workgroup's");
    constexpr int kParts = kWave / LPR, kSets = W * kParts;
    const int own = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wave = W == 1 ? 0 : own;
    const int lane = threadIdx.x & (kWave - 1), d = 4 * (lane % LPR);
    const int h = W == 1 ? 4 * blockIdx.x + own : blockIdx.x, t = blockIdx.y, b = blockIdx.z, rows = a.T * a.group;
    if (h >= a.Hq) return;
    const int hk = udiv_magic(h, a.mg_group), r = t * a.group + h - hk * a.group;
    int used;
    size_t first;
    if (a.slots) {
        const int2 i = a.info[b];
        used = i.y;
        first = static_cast<size_t>(hk) * a.slots + i.x;
    } else {
        used = (cache_keys(a, b) + a.chunk - 1) / a.chunk;
        first = (static_cast<size_t>(b) * a.Hkv + hk) * a.chunks;
    }
    if (used <= 1) return;                                           // the only chunk has written the result
    const bool in = d < a.D;
    float m = kNoScore, l = 0.0f;
    v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = wave * kParts; c0 < used; c0 += 4 * kSets) {
        v4f x[4];
        v2f st[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            x[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            st[u] = v2f{kNoScore, 0.0f};
            if (c0 + u * kSets >= used) continue;
            const size_t at = (first + min(c0 + u * kSets + lane / LPR, used - 1)) * rows + r;
            st[u] = *reinterpret_cast<const v2f*>(a.stat + at * 2);
            x[u] = *reinterpret_cast<const v4f*>(a.part + at * a.D + (in ? d : 0));
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (c0 + u * kSets + lane / LPR >= used) continue;
            const float mn = fmaxf(m, st[u][0]);
            const float f = __builtin_amdgcn_exp2f(m - mn), g = __builtin_amdgcn_exp2f(st[u][0] - mn);
            m = mn;
            l = __builtin_fmaf(l, f, st[u][1] * g);
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = __builtin_fmaf(s[e], f, x[u][e] * g);
        }
    }
    auto add = [&](float om, float ol, v4f os) {
        const float mn = fmaxf(m, om);
        const float f = __builtin_amdgcn_exp2f(m - mn), g = __builtin_amdgcn_exp2f(om - mn);
        m = mn;
        l = l * f + ol * g;
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] = s[e] * f + os[e] * g;
    };
#pragma unroll
    for (int o = LPR; o < kWave; o <<= 1) {
        const v4f os = {__shfl_xor(s[0], o, kWave), __shfl_xor(s[1], o, kWave), __shfl_xor(s[2], o, kWave), __shfl_xor(s[3], o, kWave)};
        add(__shfl_xor(m, o, kWave), __shfl_xor(l, o, kWave), os);
    }
    if constexpr (W > 1) {
        __shared__ v4f sums[W][LPR];
        __shared__ v2f stat[W];
        if (lane < LPR) sums[wave][lane] = s;
        if (lane == 0) stat[wave] = v2f{m, l};
        __syncthreads();
        if (wave != 0 || lane >= LPR) return;
#pragma unroll
        for (int w = 1; w < W; w++) add(stat[w][0], stat[w][1], sums[w][lane]);
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    if (in && lane < LPR)
        *reinterpret_cast<v2u*>(a.out + ((static_cast<size_t>(b) * a.T + t) * a.Hq + h) * a.D + d) =
            v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
}

template <int U, int RS, int KS>
constexpr int kCache4Lds = RS * KS * 16 * (Words4<U>::kRow * 4 + 8);
constexpr int kCache4MaxFound = 1024;    // sequences that find_chunk looks through (1024 of 50 to 500 keys 291 -> 202 us, 2048 599 -> 704)
constexpr int kCache4MaxChunk = 16384;   // keys of a chunk by lengths; its pages are looked up in LDS

struct Cache4Plan {
    int chunk, chunks;             // keys of a chunk; chunks of a sequence of the table's length
    int sets;                      // 16-row sets of a workgroup
    int target, least, grain, fit, slots;   // find_chunk's; slots > 0: chunks by lengths
};

// Rows of a workgroup: 16, 32, 64 or 128. A chunk has as many keys as there are rows at least (its sums are as large as its keys and values in
// 16 bits then) and 256; up to 16 rows over 512 keys, or over 1024 with heads for half the CUs, and more rows over 384 or 512, take one chunk, without a
// join. Sequences of the table's length make two workgroups per CU, or three of 64 and 128 rows. Where that makes longer chunks than the shortest (of 16 rows: than twice that),
// sequences shorter than the table would leave CUs idle: chunks go by the lengths then, for as many workgroups as the card holds at once, or twice as
// many of 16 rows, which wait for memory.
// us when this was chosen, 32 / 8 heads of 128: one token over 500 keys, in one chunk and in chunks of 256, 7.2 and 8.2 (32 sequences 8.0 and 10.6); 32 over 1000, in
// one and in two, 10.5 and 12.9 (1 over 1000 9.9 and 8.2); one over 1000, 128 keys 10.9, 256 9.3; 16 drafts over 8 x 300, in two
// and in one, 15.9 and 14.3, 4 drafts, 64 / 8 heads, over 32 x 480 21.5 and 12.8. By the table's length and by the sequences':
// one token over 16 sequences of up to 32768 64 and 60, over 128 of 2000 with tables of 8192 143 and 54, over 16 of 2000 with tables of 2048 13.8 and 15.3; 16 drafts
// over 8 sequences of 20 to 4000 25 and 17, 29, 32 / 4 heads, over 18191, 17337, 1374 and six short ones 102 and 61, 16, 32 / 4, over 119 thousand keys of 6 84 and 78.
Cache4Plan cache4_plan(int B, int T, int Hq, int Hkv, int D, long long max_keys) {
    Cache4Plan p = {};
    const int rows = T * (Hq / Hkv);
    for (p.sets = 1; 16 * p.sets < rows && p.sets < 8;) p.sets *= 2;
    const long long per_keys = static_cast<long long>(Hkv) * divup(rows, 16 * p.sets), heads = B * per_keys;
    const long long want = std::max<long long>(1, divupll((p.sets >= 4 ? 3 : 2) * default_cu_count(), heads));
    const int least = static_cast<int>(divupll(std::max(rows, 256), 128) * 128);
    const bool many = 2 * heads >= default_cu_count();
    const int one = std::max(least, p.sets == 1 ? (many ? 1024 : 512) : many ? 512 : 384);
    const long long chunk = divupll(max_keys <= one ? max_keys : std::max<long long>(divupll(max_keys, want), least), 128) * 128;
    const long long most = std::max<long long>(kCacheMaxChunk, divupll(divupll(max_keys, kGridRows), 128) * 128);
    p.chunk = static_cast<int>(std::min(chunk, most));
    p.chunks = static_cast<int>(std::max<long long>(1, divupll(max_keys, p.chunk)));
    if (p.chunks == 1 || p.chunk <= (p.sets == 1 ? 2 : 1) * least || B > kCache4MaxFound || B * max_keys > 1LL << 30) return p;
    // workgroups that a CU holds at once, by their registers (four waves, or eight for 128 rows of the widest heads)
    const int at_once = cache4_units(D) <= 4 ? (p.sets == 1 ? 3 : 2) : p.sets == 8 ? 1 : 2;
    const long long groups = static_cast<long long>(at_once) * default_cu_count() * (p.sets == 1 ? 2 : 1) / per_keys;
    p.fit = p.sets > 1 && B <= kWave;
    const long long target = std::max<long long>({1, p.fit ? groups : groups - B / 2, groups / 2, divupll(B * max_keys, kCache4MaxChunk / 2)});
    if (target + B > kGridRows) return p;
    p.target = static_cast<int>(target);
    p.least = many ? one : least;
    p.grain = p.sets >= 4 ? 64 : 128;                                // 32 keys of each of a workgroup's waves for the same rows
    p.slots = static_cast<int>(target + B);
    return p;
}

// Workspace: with slots, an int2 for each sequence (in whole 16 bytes); then the chunks' sums, then their maxima and sums of weights.
size_t cache4_parts(int B, int T, int Hq, const Cache4Plan& p) {
    return p.slots ? static_cast<size_t>(T) * Hq * p.slots : p.chunks == 1 ? 0 : static_cast<size_t>(B) * T * Hq * p.chunks;
}
size_t cache4_info_bytes(int B, const Cache4Plan& p) { return p.slots ? (static_cast<size_t>(B) * sizeof(int2) + 15) / 16 * 16 : 0; }
size_t cache4_bytes(int B, int T, int Hq, int D, const Cache4Plan& p) {
    return cache4_info_bytes(B, p) + 4 * cache4_parts(B, T, Hq, p) * (D + 2);
}

template <class T, int U, int RT, int RS, int KS>
int launch_cache4(Cache4Args a, hipStream_t s) {
    constexpr int LPR = U <= 2 ? 16 : U <= 4 ? 32 : 64;
    constexpr int kMost = kCache4Lds<U, RS, KS> + 4 * (kCache4MaxChunk / kCache4MinPage + 2);
    static_assert(kMost <= 159 * 1024, "sums and page numbers fit");
    static_assert(std::max<long long>(kCacheMaxChunk, divupll(kCacheMaxKeys, kGridRows) + 128) <= kCache4MaxChunk, "the longest chunks' pages");
    const int lds = kCache4Lds<U, RS, KS> + 4 * (((a.slots ? kCache4MaxChunk : a.chunk) >> a.page_shift) + 2);
    const int rows = a.T * (a.Hq / a.Hkv);
    a.sets = divup(rows, 16 * RT * RS);
    a.mg_sets = udiv_multiplier(a.sets);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&cache4_attention_kernel<T, U, RT, RS, KS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (attr != hipSuccess) return static_cast<int>(attr);
    // as many sequences at a time as a grid has rows
    const long long total = a.B, most = a.slots ? total : kGridRows / a.sets;
    const size_t parts = static_cast<size_t>(a.T) * a.Hq * a.chunks;     // of a sequence
    for (long long b = 0; b < total; b += most) {
        a.B = static_cast<int>(std::min(most, total - b));
        const dim3 grid(static_cast<unsigned>(a.Hkv), static_cast<unsigned>(a.slots ? a.slots : a.chunks),
                        static_cast<unsigned>(a.slots ? a.sets : a.B * a.sets));
        cache4_attention_kernel<T, U, RT, RS, KS><<<grid, 64 * RS * KS, lds, s>>>(a);
        int st = launch_status();
        if (st == FORGE_OK && (a.slots || a.chunks > 1)) {
            // a wave per row where there are few chunks: 4 x 29 rows of 14 heads, 12 chunks, 3.9 us, with four waves 4.9; 18 x 12 of 32 heads, up to 80
            // chunks, 11.2 and 8.0 (6 x 16 of 32 heads, up to 33 but most of them, 8.7 and 9.5)
            if (a.slots ? a.slots > std::max(16, 4 * a.B) : a.chunks > 16)
                cache4_join_kernel<T, LPR, 4><<<dim3(a.Hq, a.T, a.B), 256, 0, s>>>(a);
            else
                cache4_join_kernel<T, LPR, 1><<<dim3(divup(a.Hq, 4), a.T, a.B), 256, 0, s>>>(a);
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

template <class T, int U>
int launch_cache4(const Cache4Args& a, int sets, hipStream_t s) {
    if (sets == 1) return launch_cache4<T, U, 1, 1, 4>(a, s);
    if constexpr (U <= 4) {
        if (sets == 2) return launch_cache4<T, U, 2, 1, 4>(a, s);
        if (sets == 4) return launch_cache4<T, U, 2, 2, 2>(a, s);
        // twice the waves while there is a workgroup per CU at most: 4 trees of 29 drafts over 3001, 17, 0 and 2048, 14 / 2 heads of 64, 19.4 -> 16.8 us;
        // with more of them it takes from the others: 6 trees of 16 over 119 thousand keys, then 77 us, 88
        const long long groups = static_cast<long long>(a.Hkv) * divup(a.T * a.group, 128) * (a.slots ? a.slots : static_cast<long long>(a.B) * a.chunks);
        return groups <= default_cu_count() ? launch_cache4<T, U, 2, 4, 2>(a, s) : launch_cache4<T, U, 2, 4, 1>(a, s);
    } else {                                                         // (two row tiles a wave do not fit the registers)
        if (sets == 2) return launch_cache4<T, U, 1, 2, 2>(a, s);
        return sets == 4 ? launch_cache4<T, U, 1, 4, 1>(a, s) : launch_cache4<T, U, 1, 8, 1>(a, s);
    }
}

template <class T>
int launch_cache4(const Cache4Args& a, int sets, hipStream_t s) {
    switch (cache4_units(a.D)) {
    case 2: return launch_cache4<T, 2>(a, sets, s);
    case 3: return launch_cache4<T, 3>(a, sets, s);
    case 4: return launch_cache4<T, 4>(a, sets, s);
    case 6: return launch_cache4<T, 6>(a, sets, s);
    default: return launch_cache4<T, 8>(a, sets, s);
    }
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" size_t forge_cache4_attention_workspace_size(int B, int T, int Hq, int Hkv, int D, long long max_keys) {
    if (!cache_shape_ok(B, T, Hq, Hkv, D) || max_keys <= 0 || max_keys > kCacheMaxKeys) return 0;
    return cache4_bytes(B, T, Hq, D, cache4_plan(B, T, Hq, Hkv, D, max_keys));
}

extern "C" int forge_cache4_attention(const uint16_t* q, const uint8_t* cache, const int32_t* page_table, const int32_t* cache_lens,
                                      const int64_t* tree, uint16_t* out, int B, int T, int Hq, int Hkv, int D, int pages,
                                      int page_size, int table_width, float scale, int dtype, void* workspace,
                                      size_t workspace_bytes, void* stream)
{
    if (B <= 0 || T <= 0 || Hq <= 0 || D <= 0) return FORGE_OK;
    if (!cache_shape_ok(B, T, Hq, Hkv, D) || !cache4_shape_ok(Hkv, D, pages, page_size) || !q || !cache || !page_table ||
        !cache_lens || !out || table_width <= 0 || !(scale > 0.0f && scale < INFINITY) || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(cache), static_cast<const void*>(out),
                          static_cast<const void*>(workspace)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    const long long max_keys = static_cast<long long>(table_width) * page_size;
    if (max_keys > kCacheMaxKeys) return FORGE_EINVAL;
    const Cache4Plan p = cache4_plan(B, T, Hq, Hkv, D, max_keys);
    const size_t bytes = cache4_bytes(B, T, Hq, D, p), parts = cache4_parts(B, T, Hq, p);
    if (bytes && (!workspace || workspace_bytes < bytes)) return FORGE_EINVAL;
    float* part = bytes ? reinterpret_cast<float*>(static_cast<char*>(workspace) + cache4_info_bytes(B, p)) : nullptr;
    const Cache4Args a{{q, nullptr, nullptr, page_table, cache_lens, tree, out, part, part ? part + parts * D : nullptr,
                        B, T, Hq, Hkv, D, pages, __builtin_ctz(static_cast<unsigned>(page_size)), table_width,
                        p.chunk, p.chunks, Hq / Hkv, 1, udiv_multiplier(Hq / Hkv), 0u, scale},
                       cache, static_cast<int2*>(workspace), p.slots, p.target, p.least, p.grain, p.fit};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_cache4<Fp16>(a, p.sets, s) : launch_cache4<Bf16>(a, p.sets, s);
}
