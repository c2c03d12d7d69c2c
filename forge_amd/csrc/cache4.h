// The paged cache of 4 bits a value: where a head's words and numbers lie, and how words become FP16 operands.
//
// Each key or value head of D values x is held as integers n = 0..15 with a step s and a lowest value m of the
// 16-bit type: x ~ m + s n. U (2, 3, 4, 6 or 8) is the smallest with D <= 32 U; a head takes 4 U words of 8 values, the
// last ones zeros: word w holds values 8 w to 8 w + 7, of these value 2 i at bits 4 i and value 2 i + 1 at bits 16 + 4 i.
// A page's KV head is one piece of P (32 U + 8) bytes, P = page size: P rows of a key's words; the values'
// words, four positions' side by side (position / 4, word, position % 4); P times (key step, key lowest, value step,
// value lowest). So a lane of cache4_attention has 4 words of values, of 4 positions, in each of its 16-byte loads, and the U words of a key that it takes
// lie side by side (in loads of 16 bytes where U is 4 or 8, of 8 where it is 2 or 6, of 4 where it is 3); the pieces are read whole.
#pragma once

#include "float16_types.h"

namespace forge_amd {

inline int cache4_units(int D) { return D <= 64 ? 2 : D <= 96 ? 3 : D <= 128 ? 4 : D <= 192 ? 6 : 8; }
constexpr int kCache4MinPage = 16, kCache4MaxPage = 1 << 20;   // blocks of 16 positions lie in one page; 32-bit offsets in a piece

// A cache of `pages` pages is addressable: its pages' and heads' products stay in range, whatever the device's indices.
inline bool cache4_shape_ok(int Hkv, int D, int pages, int page_size) {
    return Hkv > 0 && Hkv <= 65535 && D > 0 && D % 8 == 0 && D <= 256 && pages > 0 && page_size >= kCache4MinPage && page_size <= kCache4MaxPage &&
           (page_size & (page_size - 1)) == 0 && static_cast<long long>(pages) * page_size <= 1LL << 31;
}

struct Cache4Layout {
    int U, page_shift, Hkv;
    __host__ __device__ size_t piece() const { return static_cast<size_t>(32 * U + 8) << page_shift; }
    __host__ __device__ size_t at(long long page, int hk) const { return (static_cast<size_t>(page) * Hkv + hk) * piece(); }
    // of a piece, in bytes
    __host__ __device__ uint32_t key_row(int r) const { return 16u * U * r; }
    __host__ __device__ uint32_t value_word(int r, int w) const {
        return (16u * U << page_shift) + (static_cast<uint32_t>(r >> 2) * (4 * U) + w) * 16u + (r & 3) * 4u;
    }
    __host__ __device__ uint32_t numbers(int r) const { return (32u * U << page_shift) + 8u * r; }
};

}  // namespace forge_amd
