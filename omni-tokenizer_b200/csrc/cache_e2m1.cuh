// cache_e2m1.cuh -- layout and element conversions of the 4-bit key/value cache.
//
// A cache is bytes [pages, kv_heads, page]; a page holds blocks of 16 tokens one after the
// other.  With D the head dimension rounded up to a multiple of 32 and G = D / 32 groups a
// block holds
//   keys    8 D bytes: a token's D values in their order, the first of two in a byte's low half;
//   values  8 D bytes: for each 16 columns and lane (g, c) = (lane / 4, lane % 4) of a warp one
//           word, whose bytes are columns g and g + 8 of tokens (2c, 2c + 1), then of tokens
//           (2c + 8, 2c + 9), the even token in the low half; the words of a lane lie 4
//           together (2 where D is no multiple of 64), lane after lane;
//   scales  of the keys, f16 [token % 8][group][token / 8];
//   scales  of the values, f16 [group][(token % 8) / 2][token / 8][token % 2].
// That is how the A operands of mma.sync m16n8k16 want them (tokens x columns for q k^T,
// columns x tokens for p v): a lane's values come by 16-byte loads, two of them in a byte are
// one register of the operand, and no value changes lanes.
//
// A group of 32 columns: scale = amax / 6 rounded to 6 significant bits, within [2^-14, 10752];
// value = e2m1(x / scale), to nearest even, at most 6.  e2m1 has 2 significant bits, so
// value * scale has 8 and is exact in bf16 and in f16 (hence the scale's 6 bits in its 16).  A
// group that holds a NaN or an infinity gets the scale NaN.
#pragma once
#include "e4m3.cuh"

namespace omni_b200 {

constexpr int kCacheBlock = 16, kCacheGroup = 32;
constexpr float kScaleMin = 6.103515625e-05f, kScaleMax = 10752.f; // 2^-14; 6 * 10752 is finite in f16
constexpr uint16_t kScaleNaN = 0x7e00;
__device__ __forceinline__ bool not_finite(uint16_t scale) { return (scale & 0x7c00u) == 0x7c00u; }

__host__ __device__ constexpr int cache_width(int hd) { return (hd + 31) / 32 * 32; }
template <int D> struct CacheBlock {
    static constexpr int G = D / 32;
    static constexpr int W = D % 64 == 0 ? 4 : 2; // words of a lane that lie together
    static constexpr int KEYS = 0, VALUES = 8 * D, KEY_SCALES = 16 * D, VALUE_SCALES = 16 * D + 32 * G;
    static constexpr int BYTES = 16 * D + 64 * G;
    __device__ static constexpr int key_scale(int token, int group) { return ((token % 8) * G + group) * 2 + token / 8; }
    __device__ static constexpr int value_scale(int token, int group) {
        return group * 16 + (token % 8) / 2 * 4 + token / 8 * 2 + token % 2;
    }
    // Byte of word `tile` (16 columns) of a lane.
    __device__ static constexpr int value_word(int tile, int lane) {
        return tile / W * (128 * W) + lane * (4 * W) + tile % W * 4;
    }
};
inline size_t cache_block_bytes(int hd) { return 18ull * cache_width(hd); }

// Eight values to a word, the first in the lowest bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&f)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}
// A word's eight values as four f16 pairs.
__device__ __forceinline__ void f16x8(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// The scale of a group whose largest magnitude is amax (finite, of at most 11 significant bits):
// six significant bits of amax / 6.  The product with 1/6 is within 2^-23 of it and may miss the
// middle of two scales, from which any other quotient is 2^-11 away: rounded to 16 bits first,
// it is the middle where the quotient is.
__device__ __forceinline__ float cache_scale(float amax) {
    uint32_t u = __float_as_uint(amax * (1.f / 6.f));
    u = (u + 0x80u) & ~0xffu;
    u = (u + 0x1ffffu + ((u >> 18) & 1u)) & ~0x3ffffu;
    return fminf(fmaxf(__uint_as_float(u), kScaleMin), kScaleMax);
}

// Where a cache's blocks lie.  table: [batch, table_width] pages of the sequences, or NULL:
// page b is sequence b.
struct CacheView {
    uint8_t *data;
    const int *table;
    long long page_stride, head_stride; // bytes
    int pages, page_blocks, table_width;
    // The page of block `block` of sequence b, or -1 where the table names none.
    __device__ __forceinline__ int page_of(int b, int block, int &within) const {
        const int at = block / page_blocks;
        within = block - at * page_blocks;
        const int page = table ? __ldg(table + static_cast<long long>(b) * table_width + at) : b;
        return page >= 0 && page < pages ? page : -1;
    }
    __device__ __forceinline__ uint8_t *block_at(int page, int head, int within, int block_bytes) const {
        return data + page * page_stride + head * head_stride + static_cast<long long>(within) * block_bytes;
    }
};

} // namespace omni_b200
