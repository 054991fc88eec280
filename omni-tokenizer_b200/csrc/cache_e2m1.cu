// cache_e2m1.cu -- keys and values into the 4-bit cache, and back out of it (layout and
// formulas in cache_e2m1.cuh).
//
// Both move every element once and are bound by the instructions of the conversions.  A warp
// takes the keys or the values of one block (16 tokens) of one head, so that no two warps share
// a byte: the values of tokens 2c and 2c + 1 lie in one, and a call may bring only one of the
// two.  A lane takes eight columns of a token at a time, 16 bytes, and four lanes a group, so
// that rows are read and written whole by each instruction (with 32 columns a lane, 16384 tokens
// x 8 heads of 128 were read in 22.8 us, and in 19.1 so).  Keys lie in the cache as they come;
// values change places through shared memory.
// In bf16, 8 heads of 128, in captured graphs with three sets of inputs in turn: 16384 tokens
// read in 20.1 us, 4.3 TB/s (920 instructions for a warp's 1 KB of values, ALU 74 % busy); 8191
// written in 16.3 us, 2.6 TB/s (1180 instructions, ALU 63 %), read back in 11.7, both 26.8.
#include "cache_e2m1.cuh"
#include "layer.h"

#include <algorithm>

namespace omni_b200 {
namespace {

constexpr int kWarps = 4;

struct RowsParams {
    CacheView cache;
    const int *lengths, *q_lengths;
    const void *k, *v; // written through by the read
    long long ks[3], vs[3];
    long long warps;
    int kv_heads, q_len, hd, capacity, blocks; // blocks of a sequence that a call may touch
    bool whole;
    int window, sinks;
};

// What a warp's block is: tokens [t0, t1) of sequence b, token `zero` being row 0.
struct Piece {
    int b, head, block, t0, t1;
    long long zero;
};
__device__ __forceinline__ bool piece_of(const RowsParams &p, Piece &w) {
    const uint32_t at = blockIdx.x * kWarps + (threadIdx.x >> 5); // below 2^32: the entry points see to it
    if (at >= p.warps)
        return false;
    const uint32_t of_head = at / static_cast<uint32_t>(p.kv_heads);
    w.head = static_cast<int>(at - of_head * p.kv_heads);
    w.b = static_cast<int>(of_head / static_cast<uint32_t>(p.blocks));
    const int j = static_cast<int>(of_head - static_cast<uint32_t>(w.b) * p.blocks);
    const long long n = max(p.lengths[w.b], 0);
    const long long m = p.q_lengths ? max(0, min(p.q_lengths[w.b], p.q_len)) : p.q_len;
    const long long first = p.whole ? 0 : max(n - m, 0ll);
    w.zero = p.whole ? 0 : n - m;
    const long long block = first / kCacheBlock + j, t = block * kCacheBlock;
    const long long end = min(min(t + kCacheBlock, n), static_cast<long long>(p.capacity));
    if (max(t, first) >= end) // lengths may be anything: 64 bits up to here
        return false;
    w.block = static_cast<int>(block);
    w.t0 = static_cast<int>(max(t, first));
    w.t1 = static_cast<int>(end);
    return true;
}

// Quantises eight columns, four neighbouring lanes a group: scale's f16 bits, and the word.
// Quotients in the middle of two values have to be exact, which a product with the scale's
// reciprocal is not.  It is within 2^-22 of the quotient; another quotient is at least 2^-11 of
// it away from a middle (an input has 11 significant bits, a middle times a scale 9), 2^-13 for
// the smallest middle, 1/4.  So rounding the product to multiples of 2^-14 makes middles exact
// and moves nothing else to one or across it: one addition, and its subtraction.
template <typename T> __device__ __forceinline__ uint16_t quantize_words(const Vec8<T> &in, uint32_t &word) {
    constexpr uint32_t kAbs = 0x7fff7fffu;
    uint32_t top = __vmaxu2(__vmaxu2(in.w[0].x & kAbs, in.w[0].y & kAbs), __vmaxu2(in.w[0].z & kAbs, in.w[0].w & kAbs));
    top = max(top & 0xffffu, top >> 16); // magnitudes' bits order as they do, infinities and NaN above them
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint16_t bits = static_cast<uint16_t>(top);
    const float a = to_float(*reinterpret_cast<const T *>(&bits));
    const bool finite = a <= 3.402823466e38f;
    const float scale = cache_scale(finite ? a : 0.f);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    constexpr float kGrid = 768.f; // 1.5 * 2^9: steps of 2^-14 about it
    float f[8];
    unpack8(in, f);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        ffma2(f[e], f[e + 1], f[e], f[e + 1], inv, inv, kGrid, kGrid);
        fadd2(f[e], f[e + 1], f[e], f[e + 1], -kGrid, -kGrid);
    }
    word = e2m1x8(f);
    return finite ? __half_as_ushort(__float2half_rn(scale)) : kScaleNaN;
}

// blockIdx.y: keys, or values.
template <typename T, int D> __global__ void __launch_bounds__(kWarps * 32) cache_write_kernel(const __grid_constant__ RowsParams p) {
    using B = CacheBlock<D>;
    __shared__ __align__(16) uint8_t values[kWarps][8 * D];
    Piece w;
    if (!piece_of(p, w))
        return;
    int within;
    const int page = p.cache.page_of(w.b, w.block, within);
    if (page < 0)
        return;
    const int lane = threadIdx.x & 31;
    const bool keys = blockIdx.y == 0;
    uint8_t *to = p.cache.block_at(page, w.head, within, B::BYTES), *mine = values[threadIdx.x >> 5];
    const long long *strides = keys ? p.ks : p.vs;
    const T *from = static_cast<const T *>(keys ? p.k : p.v) + w.b * strides[0] + w.head * strides[1];
    uint16_t *scales = reinterpret_cast<uint16_t *>(to + (keys ? B::KEY_SCALES : B::VALUE_SCALES));
    uint8_t *rows = keys ? to + B::KEYS : mine;
    const int base = w.block * kCacheBlock, r0 = w.t0 - base, r1 = w.t1 - base;
    constexpr int WORDS = D / 8, STEPS = kCacheBlock * WORDS / 32, AT_ONCE = STEPS < 8 ? STEPS : 8;
    const Vec8<T> none{};
    for (int i0 = 0; i0 < (r1 - r0) * WORDS; i0 += 32 * AT_ONCE) {
        Vec8<T> in[AT_ONCE];
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
            const int i = i0 + 32 * x + lane, r = r0 + i / WORDS, col = i % WORDS * 8;
            in[x] = r < r1 && col < p.hd ? load8(from + (base + r - w.zero) * strides[2] + col) : none;
        }
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
            if (i0 + 32 * x >= (r1 - r0) * WORDS)
                break; // the same for all lanes
            const int i = i0 + 32 * x + lane, r = r0 + i / WORDS, c = i % WORDS;
            uint32_t word;
            const uint16_t scale = quantize_words(in[x], word);
            if (r < r1) {
                *reinterpret_cast<uint32_t *>(rows + r * (D / 2) + c * 4) = word;
                if (c % 4 == 0)
                    scales[keys ? B::key_scale(r, c / 4) : B::value_scale(r, c / 4)] = scale;
            }
        }
    }
    if (keys)
        return;
    __syncwarp();
    // Words of the values: columns g and g + 8 of tokens 2c, 2c + 1, 2c + 8 and 2c + 9.
    const int g = lane >> 2, c = lane & 3;
    uint32_t keep = 0; // bits of tokens that this call does not bring
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const int t = 2 * c + 8 * half + odd;
            if (t < r0 || t >= r1)
                keep |= 0x0f0fu << (16 * half + 4 * odd);
        }
    // Of two tokens' rows of eight columns: bytes with both tokens of columns g % 2, g % 2 + 2, ...
    const int right = g & 1 ? 4 : 0, left = 4 - right;
    auto both = [&](uint32_t even, uint32_t odd) { return ((even >> right) & 0x0f0f0f0fu) | ((odd << left) & 0xf0f0f0f0u); };
    const uint32_t pick = (g >> 1) | (4 + (g >> 1)) << 4; // byte g / 2 of two words
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        uint2 row[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            row[e] = *reinterpret_cast<const uint2 *>(mine + (2 * c + 8 * (e >> 1) + (e & 1)) * (D / 2) + x * 8);
        const uint32_t low = __byte_perm(both(row[0].x, row[1].x), both(row[0].y, row[1].y), pick);
        const uint32_t high = __byte_perm(both(row[2].x, row[3].x), both(row[2].y, row[3].y), pick);
        uint32_t word = __byte_perm(low, high, 0x5410);
        uint32_t *at = reinterpret_cast<uint32_t *>(to + B::VALUES + B::value_word(x, lane));
        if (keep)
            word = (word & ~keep) | (*at & keep);
        *at = word;
    }
}

// Stores eight columns, f16 pairs, times their scale.
template <typename T> __device__ __forceinline__ void store_columns(T *y, const uint32_t (&h)[4], uint16_t scale) {
    const float s = __half2float(__ushort_as_half(scale));
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&h[e]));
        fmul2(f[2 * e], f[2 * e + 1], two.x, two.y, s, s);
    }
    store8(y, pack8<T>(f));
}

// blockIdx.y: keys, or values.  WHOLE: for prompts, where what is not finite must not stand among
// the values (0 * NaN would reach queries that do not see it): they get zeros there, and the
// token's keys NaN, which a mask hides.
template <typename T, int D, bool WHOLE> __global__ void __launch_bounds__(kWarps * 32) cache_read_kernel(const __grid_constant__ RowsParams p) {
    using B = CacheBlock<D>;
    __shared__ __align__(16) uint8_t values[kWarps][8 * D];
    Piece w;
    if (!piece_of(p, w))
        return;
    const int base = w.block * kCacheBlock;
    if (WHOLE && p.window > 0) { // keys that no query of a prompt sees, nor stand near one that is seen
        const long long n = min(max(p.lengths[w.b], 0), p.capacity);
        const long long m = p.q_lengths ? max(0, min(p.q_lengths[w.b], p.q_len)) : p.q_len;
        if (base + kCacheBlock <= n - m - p.window - 127 && base >= p.sinks + 128ll)
            return;
    }
    const int lane = threadIdx.x & 31;
    const bool keys = blockIdx.y == 0;
    int within;
    const int page = p.cache.page_of(w.b, w.block, within);
    const long long *strides = keys ? p.ks : p.vs;
    T *to = static_cast<T *>(const_cast<void *>(keys ? p.k : p.v)) + w.b * strides[0] + w.head * strides[1];
    const uint8_t *from = page < 0 ? nullptr : p.cache.block_at(page, w.head, within, B::BYTES);
    const int r0 = w.t0 - base, r1 = w.t1 - base;
    constexpr int WORDS = D / 8, STEPS = kCacheBlock * WORDS / 32;
    uint8_t *mine = values[threadIdx.x >> 5];
    if (from && !keys) {
#pragma unroll
        for (int i = lane; i < 8 * D / 16; i += 32)
            reinterpret_cast<uint4 *>(mine)[i] = reinterpret_cast<const uint4 *>(from + B::VALUES)[i];
    }
    __syncwarp();
    // All of a warp's reads, then its writes.  Keys: a word a step.  Values: eight bytes, each
    // the column's nibbles of two tokens.
    uint32_t words[STEPS][2] = {};
    uint16_t scales[STEPS], value_scales[B::G] = {};
    if (WHOLE && keys && from && lane < kCacheBlock)
#pragma unroll
        for (int g = 0; g < B::G; ++g)
            value_scales[g] = *reinterpret_cast<const uint16_t *>(from + B::VALUE_SCALES + 2 * B::value_scale(lane, g));
#pragma unroll
    for (int x = 0; x < STEPS; ++x) {
        const int i = 32 * x + lane, r = r0 + i / WORDS, c = i % WORDS;
        scales[x] = WHOLE && !keys ? 0 : kScaleNaN; // a page that the cache does not have reads as NaN
        if (!from || r >= r1)
            continue;
        if (keys) {
            words[x][0] = *reinterpret_cast<const uint32_t *>(from + B::KEYS + r * (D / 2) + c * 4);
            scales[x] = *reinterpret_cast<const uint16_t *>(from + B::KEY_SCALES + 2 * B::key_scale(r, c / 4));
        } else {
            scales[x] = *reinterpret_cast<const uint16_t *>(from + B::VALUE_SCALES + 2 * B::value_scale(r, c / 4));
            if (WHOLE && not_finite(scales[x]))
                scales[x] = 0;
            const uint8_t *at = mine + B::value_word(c / 2, r % 8 / 2) + r / 8 * 2 + c % 2;
            uint32_t b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) // columns 8 c + e, of lane 4 e + (r % 8) / 2
                b[e] = at[16 * B::W * e];
#pragma unroll
            for (int h = 0; h < 2; ++h) // nibbles of two columns in bytes 0 and 2
                words[x][h] = __byte_perm(__byte_perm(b[4 * h], b[4 * h + 1], 0x0040), __byte_perm(b[4 * h + 2], b[4 * h + 3], 0x0040), 0x5410);
        }
    }
    uint32_t lost = 0; // tokens of which some value is not finite
    if (WHOLE && keys && from) {
        bool mine = false;
#pragma unroll
        for (int g = 0; g < B::G; ++g)
            mine |= not_finite(value_scales[g]);
        lost = __ballot_sync(0xffffffffu, mine);
    }
#pragma unroll
    for (int x = 0; x < STEPS; ++x) {
        const int i = 32 * x + lane, r = r0 + i / WORDS, c = i % WORDS;
        if (r >= r1 || c * 8 >= p.hd)
            continue;
        uint32_t h[4];
        if (keys) {
            f16x8(words[x][0], h);
            if (lost >> r & 1u)
                scales[x] = kScaleNaN;
        } else {
            uint32_t two[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t w = (words[x][e] >> (r % 2 * 4)) & 0x0f0f0f0fu;
                w |= w >> 4;
                f16x8(w, two);
                h[2 * e] = two[0];
                h[2 * e + 1] = two[2];
            }
        }
        store_columns(to + (base + r - w.zero) * strides[2] + c * 8, h, scales[x]);
    }
}

RowsParams rows_params(const CacheArgs &c, const void *k, const void *v, const long long (&ks)[3], const long long (&vs)[3]) {
    RowsParams p{};
    p.cache.data = static_cast<uint8_t *>(c.data);
    p.cache.table = c.table;
    p.cache.page_stride = c.page_stride;
    p.cache.head_stride = c.head_stride;
    p.cache.pages = c.pages;
    p.cache.page_blocks = c.page_tokens / kCacheBlock;
    p.cache.table_width = c.table_width;
    p.lengths = c.lengths;
    p.q_lengths = c.q_lengths;
    p.k = k;
    p.v = v;
    for (int d = 0; d < 3; ++d) {
        p.ks[d] = ks[d];
        p.vs[d] = vs[d];
    }
    p.kv_heads = c.kv_heads;
    p.q_len = c.q_len;
    p.hd = c.hd;
    p.capacity = static_cast<int>(c.capacity());
    // q_len tokens that may begin inside a block.
    p.blocks = static_cast<int>(std::min<long long>((c.q_len + 14ll) / kCacheBlock + 1, c.capacity() / kCacheBlock));
    return p;
}

template <typename T, int D> int launch_rows(RowsParams &p, int batch, bool read, cudaStream_t stream) {
    p.warps = static_cast<long long>(batch) * p.blocks * p.kv_heads;
    const long long ctas = (p.warps + kWarps - 1) / kWarps;
    if (ctas > 0x7fffffffll)
        return static_cast<int>(cudaErrorInvalidValue);
    const dim3 grid(static_cast<unsigned>(ctas), 2);
    if (read && !p.whole)
        cache_read_kernel<T, D, false><<<grid, kWarps * 32, 0, stream>>>(p);
    else if constexpr (sizeof(T) == 2) {
        if (read)
            cache_read_kernel<T, D, true><<<grid, kWarps * 32, 0, stream>>>(p);
        else
            cache_write_kernel<T, D><<<grid, kWarps * 32, 0, stream>>>(p);
    }
    return static_cast<int>(cudaGetLastError());
}
template <typename T> int launch_width(RowsParams &p, int batch, bool read, cudaStream_t stream) {
    switch (cache_width(p.hd)) {
    case 32:
        return launch_rows<T, 32>(p, batch, read, stream);
    case 64:
        return launch_rows<T, 64>(p, batch, read, stream);
    case 96:
        return launch_rows<T, 96>(p, batch, read, stream);
    default:
        return launch_rows<T, 128>(p, batch, read, stream);
    }
}

} // namespace

int cache_write_launch(const CacheArgs &c, const void *k, const void *v, const long long (&ks)[3],
                       const long long (&vs)[3], int dtype, cudaStream_t stream) {
    RowsParams p = rows_params(c, k, v, ks, vs);
    return dtype == kBF16 ? launch_width<__nv_bfloat16>(p, c.batch, false, stream)
                          : launch_width<__half>(p, c.batch, false, stream);
}

int cache_read_launch(const CacheArgs &c, void *k, void *v, const long long (&ks)[3], const long long (&vs)[3],
                      int dtype, const CacheReadRange &range, cudaStream_t stream) {
    RowsParams p = rows_params(c, k, v, ks, vs);
    if (range.whole) {
        p.whole = true;
        p.capacity = range.kv_len;
        p.blocks = (range.kv_len + kCacheBlock - 1) / kCacheBlock;
        p.window = range.window;
        p.sinks = range.sinks;
    }
    if (dtype == kF32)
        return launch_width<float>(p, c.batch, true, stream);
    return dtype == kBF16 ? launch_width<__nv_bfloat16>(p, c.batch, true, stream)
                          : launch_width<__half>(p, c.batch, true, stream);
}

} // namespace omni_b200
