// cache_e2m1.cu -- keys and values into the 4-bit cache, and back out of it (layout and
// formulas in cache_e2m1.cuh).
//
// Both move every element once and are bound by the memory's traffic.  A warp takes one
// block (16 tokens) of one head, so that no two warps share a byte: the values of tokens 2c
// and 2c + 1 lie in one, and a call may bring only one of the two.  A lane takes groups of
// 32 columns of a token, whole: its largest magnitude needs no other lane, and its 64 bytes
// are two memory sectors.  Keys lie in the cache as they come; values change places
// through shared memory.
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
    const long long at = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (at >= p.warps)
        return false;
    const long long of_head = at / p.kv_heads;
    w.head = static_cast<int>(at - of_head * p.kv_heads);
    w.b = static_cast<int>(of_head / p.blocks);
    const int j = static_cast<int>(of_head - static_cast<long long>(w.b) * p.blocks);
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

__device__ __forceinline__ uint32_t abs_bits(uint32_t pair) { return pair & 0x7fff7fffu; }

// Quantises 32 columns (those behind `cols` are zeros): scale's f16 bits, and values in q.
template <typename T> __device__ __forceinline__ uint16_t quantize_group(const T *x, int cols, uint4 &q) {
    Vec8<T> in[4];
    uint32_t top2 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        in[i].w[0] = make_uint4(0u, 0u, 0u, 0u);
        if (i * 8 < cols)
            in[i] = load8(x + i * 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = __vmaxu2(__vmaxu2(abs_bits(in[i].w[0].x), abs_bits(in[i].w[0].y)),
                                    __vmaxu2(abs_bits(in[i].w[0].z), abs_bits(in[i].w[0].w)));
        top2 = __vmaxu2(top2, m);
    }
    // Magnitudes' bits order as the magnitudes do, infinities and NaN above them.
    const uint16_t top = static_cast<uint16_t>(max(top2 & 0xffffu, top2 >> 16));
    T amax;
    *reinterpret_cast<uint16_t *>(&amax) = top;
    const float a = to_float(amax);
    const bool finite = a <= 3.402823466e38f;
    const float scale = cache_scale(finite ? a : 0.f);
    const Divisor d = divisor_of(scale);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float f[8];
        unpack8(in[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) // exact quotients: 16-bit inputs meet the middle of two values
            f[e] = d.quotient<true>(f[e]);
        w[i] = e2m1x8(f);
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
    return finite ? __half_as_ushort(__float2half_rn(scale)) : kScaleNaN;
}

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
    uint8_t *to = p.cache.block_at(page, w.head, within, B::BYTES), *mine = values[threadIdx.x >> 5];
    const T *k = static_cast<const T *>(p.k) + w.b * p.ks[0] + w.head * p.ks[1];
    const T *v = static_cast<const T *>(p.v) + w.b * p.vs[0] + w.head * p.vs[1];
    uint16_t *k_scales = reinterpret_cast<uint16_t *>(to + B::KEY_SCALES);
    uint16_t *v_scales = reinterpret_cast<uint16_t *>(to + B::VALUE_SCALES);
    const int base = w.block * kCacheBlock, r0 = w.t0 - base, r1 = w.t1 - base;
    for (int i = lane; i < (r1 - r0) * B::G; i += 32) {
        const int r = r0 + i / B::G, g = i % B::G;
        const long long row = base + r - w.zero;
        uint4 q;
        k_scales[B::key_scale(r, g)] = quantize_group(k + row * p.ks[2] + g * 32, p.hd - g * 32, q);
        *reinterpret_cast<uint4 *>(to + B::KEYS + r * (D / 2) + g * 16) = q;
        v_scales[B::value_scale(r, g)] = quantize_group(v + row * p.vs[2] + g * 32, p.hd - g * 32, q);
        *reinterpret_cast<uint4 *>(mine + r * (D / 2) + g * 16) = q;
    }
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
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        uint32_t word = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const int t = 2 * c + 8 * half + odd;
                const uint2 row = *reinterpret_cast<const uint2 *>(mine + t * (D / 2) + x * 8);
                word |= (((row.x >> (4 * g)) & 15u) | ((row.y >> (4 * g)) & 15u) << 8) << (16 * half + 4 * odd);
            }
        uint32_t *at = reinterpret_cast<uint32_t *>(to + B::VALUES + B::value_word(x, lane));
        *at = keep ? (word & ~keep) | (*at & keep) : word;
    }
}

// Stores 32 columns of a token, as many as there are.
template <typename T> __device__ __forceinline__ void store_group(T *y, int cols, const uint4 &q, uint16_t scale) {
    const float s = __half2float(__ushort_as_half(scale));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[4];
        f16x8(w[i], h);
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&h[e]));
            f[2 * e] = two.x * s;
            f[2 * e + 1] = two.y * s;
        }
        if (i * 8 < cols)
            store8(y + i * 8, pack8<T>(f));
    }
}

template <typename T, int D> __global__ void __launch_bounds__(kWarps * 32) cache_read_kernel(const __grid_constant__ RowsParams p) {
    using B = CacheBlock<D>;
    __shared__ __align__(16) uint8_t values[kWarps][8 * D];
    Piece w;
    if (!piece_of(p, w))
        return;
    const int base = w.block * kCacheBlock;
    if (p.window > 0) { // keys that no query of a prompt sees, nor stand near one that is seen
        const long long n = min(max(p.lengths[w.b], 0), p.capacity);
        const long long m = p.q_lengths ? max(0, min(p.q_lengths[w.b], p.q_len)) : p.q_len;
        if (base + kCacheBlock <= n - m - p.window - 127 && base >= p.sinks + 128ll)
            return;
    }
    const int lane = threadIdx.x & 31;
    int within;
    const int page = p.cache.page_of(w.b, w.block, within);
    T *k = static_cast<T *>(const_cast<void *>(p.k)) + w.b * p.ks[0] + w.head * p.ks[1];
    T *v = static_cast<T *>(const_cast<void *>(p.v)) + w.b * p.vs[0] + w.head * p.vs[1];
    const uint8_t *from = page < 0 ? nullptr : p.cache.block_at(page, w.head, within, B::BYTES);
    uint8_t *mine = values[threadIdx.x >> 5];
    if (from)
        for (int i = lane; i < 8 * D / 16; i += 32)
            reinterpret_cast<uint4 *>(mine)[i] = reinterpret_cast<const uint4 *>(from + B::VALUES)[i];
    __syncwarp();
    const int r0 = w.t0 - base, r1 = w.t1 - base;
    for (int i = lane; i < (r1 - r0) * B::G; i += 32) {
        const int r = r0 + i / B::G, g = i % B::G;
        const long long row = base + r - w.zero;
        uint16_t ks = kScaleNaN, vs = kScaleNaN; // a page that the cache does not have reads as NaN
        uint4 q = make_uint4(0u, 0u, 0u, 0u), u = q;
        if (from) {
            ks = *reinterpret_cast<const uint16_t *>(from + B::KEY_SCALES + 2 * B::key_scale(r, g));
            vs = *reinterpret_cast<const uint16_t *>(from + B::VALUE_SCALES + 2 * B::value_scale(r, g));
            q = *reinterpret_cast<const uint4 *>(from + B::KEYS + r * (D / 2) + g * 16);
            uint32_t word[4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t low = 0, high = 0; // columns 0 to 7 and 8 to 15 of the 16
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int from_lane = 4 * e + (r % 8) / 2;
                    const uint32_t two = *reinterpret_cast<const uint16_t *>(mine + B::value_word(2 * g + x, from_lane) + r / 8 * 2);
                    low |= ((two >> (r % 2 * 4)) & 15u) << (4 * e);
                    high |= ((two >> (8 + r % 2 * 4)) & 15u) << (4 * e);
                }
                word[2 * x] = low;
                word[2 * x + 1] = high;
            }
            u = make_uint4(word[0], word[1], word[2], word[3]);
        }
        store_group(k + row * p.ks[2] + g * 32, p.hd - g * 32, q, ks);
        store_group(v + row * p.vs[2] + g * 32, p.hd - g * 32, u, vs);
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
    if (read)
        cache_read_kernel<T, D><<<static_cast<unsigned>(ctas), kWarps * 32, 0, stream>>>(p);
    else if constexpr (sizeof(T) == 2)
        cache_write_kernel<T, D><<<static_cast<unsigned>(ctas), kWarps * 32, 0, stream>>>(p);
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
