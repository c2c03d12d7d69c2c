// Attention over whole prompts packed without padding: softmax(scale Q K^T) V within each sequence, causal
// or not, with grouped heads.
//
// A workgroup of RS x KS waves takes 32 RS query rows of one sequence and head, a wave 32 of them (attn_tile.h)
// and 64 keys of each tile of 64 KS, which all waves share: K and V rows come by LDS DMA into NS buffers each,
// the next tiles' while this one is multiplied, one barrier a tile. Tiles past the diagonal are not
// loaded, only those that cross it are masked.
//
// Bound: the softmax, whose vector instructions wait for each tile's maximum and which the other wave of a SIMD does not cover (matrix
// units busy 42 to 53 %), at the clock that the matrix units leave (1.6 to 1.7 GHz). Causal, 32 / 8 heads of 128: a prompt of
// 4096 150 to 162 us by box (850 to 915 TFLOP/s), of 9001 + 5120 + 2263 859 to 917 (1003 to 1071). Two workgroups of 4 waves a CU;
// 8 waves that share their tiles measured the same.
//
// The grid is laid out without reading cu_seqlens on the host: sequence b's tiles start at
// cu[b] / rows + b, which leaves room for each sequence's last partial tile.
#include "attn_tile.h"
#include "ring_tile.h"

#include <climits>

namespace forge_amd {

struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    const int32_t* cu;
    long long q_token, q_head, k_token, k_head, v_token, v_head;
    int sequences, tokens, Hq, Hkv, D, tiles, group;
    uint32_t mg_group, mg_hkv;   // udiv_magic multipliers
    float scale;
};

constexpr int kPromptKeys = 64;

template <class T, int DP, int RS, int KS, int NS, bool CAUSAL>
__global__ __launch_bounds__(64 * RS * KS, DP > 128 ? 1 : 2) void prompt_attention_kernel(PromptArgs a)
{
    using Rows = KvRows<DP>;
    constexpr int W = RS * KS, kRows = 32 * RS, kKeys = kPromptKeys * KS, kTile = kKeys * Rows::kBytes;
    constexpr int kIns = kKeys * Rows::kChunks / kWave / W;   // DMA instructions per wave, tile and tensor
    static_assert(kKeys * Rows::kChunks % (kWave * W) == 0, "a tile splits evenly over the waves");
    extern __shared__ __align__(1024) int8_t lds[];                 // K, V of buffer 0, then of buffer 1 ...

    const int group = a.group;
    // Query tiles from the last (the longest in a causal prompt) on; units (tile, KV head) go round
    // the 8 XCDs, whose workgroups are dealt in turn, so that the heads of a group meet in one L2.
    const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
    const int ig = udiv_magic(i, a.mg_group), unit = ig * 8 + xcd, tile = udiv_magic(unit, a.mg_hkv);
    const int hk = unit - tile * a.Hkv, hq = hk * group + i - ig * group;
    const int id = a.tiles - 1 - tile;
    if (id < 0) return;

    auto cu = [&](int b) { return min(max(a.cu[b], 0), a.tokens); };
    int b = 0;                                                       // the last b whose first tile is <= id,
    for (int span = a.sequences + 1; span > 1;) {                    // 64 candidates at a time
        const int step = (span + 63) / 64, c = b + static_cast<int>(threadIdx.x & (kWave - 1)) * step;
        const bool on = c < min(b + span, a.sequences + 1) && cu(c) / kRows + c <= id;
        b += max(__popcll(__ballot(on)) - 1, 0) * step;
        span = step;
    }
    b = __builtin_amdgcn_readfirstlane(min(b, a.sequences));
    const int start = cu(b);
    const int len = (b < a.sequences ? cu(b + 1) : a.tokens) - start;
    const int row0 = (id - (start / kRows + b)) * kRows;
    if (row0 < 0 || row0 >= len) return;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x & (kWave - 1);
    const int rs = wave / KS, ks = wave % KS, row = row0 + 32 * rs + (lane & 31);
    uint16_t* out = a.out + (static_cast<size_t>(start + row) * a.Hq + hq) * a.D;
    if (b == a.sequences) {                                          // rows after the last sequence
        for (int d = 4 * (lane >> 5); d < a.D; d += 8)
            if (row < len && ks == 0) *reinterpret_cast<v2u*>(out + d) = v2u{0u, 0u};
        return;
    }

    AttnWave<T, DP, kPromptKeys / 32> w;
    w.init();
    w.keys(len);
    w.load_q(a.q + static_cast<size_t>(start + row) * a.q_token + hq * a.q_head, row < len, a.D);

    const uint16_t* kbase = a.k + static_cast<size_t>(start) * a.k_token + hk * a.k_head;
    const uint16_t* vbase = a.v + static_cast<size_t>(start) * a.v_token + hk * a.v_head;
    int dma_row[kIns];
    uint32_t koff[kIns], voff[kIns];
#pragma unroll
    for (int n = 0; n < kIns; n++) {
        const int c = (wave * kIns + n) * kWave + lane, r = c / Rows::kChunks, p = c % Rows::kChunks;
        const int ck = p ^ Rows::swz_k(r), cv = p ^ Rows::swz_v(r);
        dma_row[n] = r;
        koff[n] = 8 * ck < a.D ? static_cast<uint32_t>(r * a.k_token * 2 + 16 * ck) : kOutOfRange;
        voff[n] = 8 * cv < a.D ? static_cast<uint32_t>(r * a.v_token * 2 + 16 * cv) : kOutOfRange;
    }
    const int end = CAUSAL ? min(row0 + kRows, len) : len;
    const int tiles = (end + kKeys - 1) / kKeys;
    const uint32_t lds0 = lds_address(lds);
    // rows past the sequence's end read as zeros
    auto load = [&](int t) {
        const int left = len - t * kKeys;
        const v4i kr = row_rsrc(kbase + static_cast<size_t>(t) * kKeys * a.k_token,
                                static_cast<uint32_t>((kKeys - 1) * a.k_token * 2 + 2 * a.D));
        const v4i vr = row_rsrc(vbase + static_cast<size_t>(t) * kKeys * a.v_token,
                                static_cast<uint32_t>((kKeys - 1) * a.v_token * 2 + 2 * a.D));
        const uint32_t to = lds0 + (t % NS) * 2 * kTile;
#pragma unroll
        for (int n = 0; n < kIns; n++)
            dma16_rows(kr, dma_row[n] < left ? koff[n] : kOutOfRange, to + (wave * kIns + n) * 1024);
#pragma unroll
        for (int n = 0; n < kIns; n++)
            dma16_rows(vr, dma_row[n] < left ? voff[n] : kOutOfRange, to + kTile + (wave * kIns + n) * 1024);
    };
    const float scale2 = a.scale * 1.44269504f;
    const int first = row0 + 32 * rs, ahead = first - kPromptKeys * ks;
    // tiles that reach this wave's rows
    const int mine = !CAUSAL ? tiles : ahead < 0 ? 0 : min(tiles, ahead / kKeys + 1);
    __shared__ int odd;
    if (threadIdx.x == 0) odd = -1;
    auto seen = [&](int t) {
        return [&, k0 = t * kKeys + kPromptKeys * ks](int kb) { return bits_to((CAUSAL ? min(row, len - 1) : len - 1) - k0 - 32 * kb); };
    };
    auto next = [&](int t) {
        if (t + NS - 1 <= tiles) wait_vm_lgkm<2 * kIns*(NS - 2)>();
        else wait_vm_lgkm<0>();
        lds_barrier();                                               // tile t is whole, tile t - 1 is read
        if (t + NS - 1 < tiles) load(t + NS - 1);
        if (CAUSAL && (t + 1) * kKeys - 1 > row0) {                  // rows see it in part (what lies past the end is zeros)
            int8_t* v = lds + (t % NS) * 2 * kTile + kTile;
            w.template take_odd_values<W, KS>(v, v + kPromptKeys * ks * Rows::kBytes, wave, t, &odd, seen(t));
        }
    };
#pragma unroll
    for (int t = 0; t < NS - 1; t++)
        if (t < tiles) load(t);
    int t = 0;
    for (; t < mine; t++) {
        next(t);
        const int8_t* at = lds + (t % NS) * 2 * kTile + kPromptKeys * ks * Rows::kBytes;
        const int k0 = t * kKeys + kPromptKeys * ks;
        v16f s[kPromptKeys / 32];
        w.scores(at, s);
        w.finish(s, at + kTile, scale2, t == 0, (CAUSAL && k0 + kPromptKeys - 1 > first) || k0 + kPromptKeys > len, seen(t));
    }
    for (; t < tiles; t++) next(t);
    const bool live = row < len;
    if constexpr (KS == 1) {
        const float l = half_sum(w.l);
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        if (!live) return;
#pragma unroll
        for (int j = 0; j < DP / 32; j++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int d = 32 * j + 2 * e + 4 * (lane >> 5);
                if (d < a.D)
                    *reinterpret_cast<v2u*>(out + d) = v2u{T::pack(w.o[j][e] * inv, w.o[j][e + 1] * inv),
                                                           T::pack(w.o[j][e + 2] * inv, w.o[j][e + 3] * inv)};
            }
    } else {
        auto* sh = reinterpret_cast<typename AttnWave<T, DP, kPromptKeys / 32>::template Shared<W>*>(lds);
        wait_vm_lgkm<0>();
        __syncthreads();
        w.leave(sh, wave, live);
        __syncthreads();
        if (!live) return;
        w.template join<KS>(sh, wave, [&](int j, int e, v4f s, float, float sum) {
            const int d = 32 * j + 8 * e + 4 * (lane >> 5);
            if (d >= a.D) return;
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            *reinterpret_cast<v2u*>(out + d) = v2u{T::pack(s[0] * inv, s[1] * inv), T::pack(s[2] * inv, s[3] * inv)};
        });
    }
}

template <class T, int DP, int RS, int KS, int NS, bool CAUSAL>
int launch_prompt(PromptArgs a, hipStream_t s) {
    constexpr int kTiles = NS * 2 * kPromptKeys * KS * KvRows<DP>::kBytes, kSums = KS > 1 ? sizeof(typename AttnWave<T, DP, 2>::template Shared<RS * KS>) : 0;
    constexpr int kLds = kTiles > kSums ? kTiles : kSums;
    const long long tiles = a.tokens / (32 * RS) + static_cast<long long>(a.sequences) + 1;
    const long long units = tiles * a.Hkv, wgs = divupll(units, 8) * 8 * (a.Hq / a.Hkv);
    // udiv_magic's range; 2^31 / 65536 tiles of heads at least
    if ((units + 8) * a.Hkv >= 1LL << 32 || wgs * a.group >= 1LL << 32 || wgs > INT_MAX) return FORGE_EINVAL;
    a.mg_group = udiv_multiplier(a.group);
    a.mg_hkv = udiv_multiplier(a.Hkv);
    a.tiles = static_cast<int>(tiles);
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&prompt_attention_kernel<T, DP, RS, KS, NS, CAUSAL>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return static_cast<int>(attr);
    prompt_attention_kernel<T, DP, RS, KS, NS, CAUSAL><<<static_cast<unsigned>(wgs), 64 * RS * KS, kLds, s>>>(a);
    return launch_status();
}

template <class T, int DP, int RS, int KS, int NS>
int launch_prompt(const PromptArgs& a, bool causal, hipStream_t s) {
    return causal ? launch_prompt<T, DP, RS, KS, NS, true>(a, s) : launch_prompt<T, DP, RS, KS, NS, false>(a, s);
}

// While workgroups of 128 rows are fewer than the CUs, the time is that of the longest sequence's chain of
// tiles: 64 rows a workgroup then, and two waves for each 32 that take 64 keys each of a tile. us, 128 rows /
// 64, heads of 64: 16 heads of 512 tokens 11.3 / 9.0, 1024 19.1 / 13.6, 2048 34.7 / 27.4; 32 heads of 2048 (544
// workgroups) 39.7 / 51.4; 64 tokens 4.7 / 5.7.
template <class T>
int launch_prompt(const PromptArgs& a, bool causal, hipStream_t s) {
    const bool few = a.tokens >= 256 && (a.tokens / 128 + static_cast<long long>(a.sequences)) * a.Hq < default_cu_count();
    if (a.D <= 64) return few ? launch_prompt<T, 64, 2, 2, 3>(a, causal, s) : launch_prompt<T, 64, 4, 1, 4>(a, causal, s);
    if (a.D <= 96) return few ? launch_prompt<T, 96, 2, 2, 2>(a, causal, s) : launch_prompt<T, 96, 4, 1, 3>(a, causal, s);
    if (a.D <= 128) return few ? launch_prompt<T, 128, 2, 2, 2>(a, causal, s) : launch_prompt<T, 128, 4, 1, 2>(a, causal, s);
    return launch_prompt<T, 256, 4, 1, 2>(a, causal, s);
}

}  // namespace forge_amd

using namespace forge_amd;

extern "C" int forge_prompt_attention(const uint16_t* q, const uint16_t* k, const uint16_t* v, const int32_t* cu_seqlens,
                                      uint16_t* out, int sequences, int tokens, int Hq, int Hkv, int D,
                                      long long q_token, long long q_head, long long k_token, long long k_head,
                                      long long v_token, long long v_head, float scale, int causal, int dtype,
                                      void* stream)
{
    if (sequences <= 0 || tokens <= 0 || Hq <= 0 || D <= 0) return FORGE_OK;
    if (!q || !k || !v || !cu_seqlens || !out || Hkv <= 0 || Hq % Hkv != 0 || D % 8 != 0 || D > 256 ||
        !(scale > 0.0f && scale < INFINITY) || (dtype != FORGE_FP16 && dtype != FORGE_BF16))
        return FORGE_EINVAL;
    for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k), static_cast<const void*>(v),
                          static_cast<const void*>(out)})
        if (!aligned(p, 16)) return FORGE_EINVAL;
    // a tile's rows, 128 at most, are addressed in 31 bits
    for (long long st : {q_token, q_head, k_token, k_head, v_token, v_head})
        if (st < 0 || st % 8 != 0 || st > (1 << 23)) return FORGE_EINVAL;
    const PromptArgs a{q, k, v, out, cu_seqlens, q_token, q_head, k_token, k_head, v_token, v_head,
                       sequences, tokens, Hq, Hkv, D, 0, Hq / Hkv, 0u, 0u, scale};
    hipStream_t s = as_stream(stream);
    return dtype == FORGE_FP16 ? launch_prompt<Fp16>(a, causal != 0, s) : launch_prompt<Bf16>(a, causal != 0, s);
}
