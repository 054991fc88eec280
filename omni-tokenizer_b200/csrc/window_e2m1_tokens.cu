// window_e2m1_tokens.cu -- sliding-window attention over the 4-bit cache for few queries:
// the next tokens of sequences (layout of the cache in cache_e2m1.cuh).
//
// softmax(scale * q k^T + mask) v for the `group * q_len` query rows that share a key head,
// 8 NT of them at a time as the COLUMNS of mma.sync m16n8k16: keys (16 tokens x 16 columns)
// and values (16 columns x 16 tokens) are the A operands, so that what has to be converted
// goes through the tensor cores once for all rows, and rows fill up in steps of 8.
//   S^T = K q^T: a lane has tokens g and g + 8 (g = lane / 4) of queries 2c and 2c + 1
//     (c = lane % 4); the sum over a head's columns may go in any order, so lane c takes the
//     columns that lie together in its words.
//   O^T = V^T P^T: P^T's B operand is S^T's accumulators packed to f16 and turned by
//     movmatrix.
// Every product is f16 x f16 with fp32 sums whatever q's type is: the cache's values are
// exact in f16, P <= 2^8 is rounded to 11 bits there (bf16: 8), and a bf16 row of q is
// multiplied by the power of two that brings its largest element to [2^14, 2^15): elements
// down to 2^-28 of it keep all their bits, what is below loses less than 2^-39 of it.
//
// The bound is the cache's bytes.  A block of 16 tokens of a head (2304 bytes at 128 columns)
// is one contiguous piece; each warp copies its own blocks to a ring in shared memory
// (cp.async, no barrier between warps) and keeps its own softmax state.  The running maximum
// is lazy: a warp looks at the other lanes' maxima only when some score is more than 2^8
// above the reference.  A cluster of CTAs splits the keys of one tile of rows; the parts meet
// in distributed shared memory, in rank order (no atomics).
#include "cache_e2m1.cuh"
#include "fmha.h"
#include "layer.h"

#include <algorithm>
#include <cmath>

namespace omni_b200 {
namespace {

constexpr int kWarps = 4, kMaxParts = 16;
constexpr float kLazy = 8.f; // log2 units a score may be above the reference

struct TokensParams {
    CacheView cache;
    const uint16_t *q;
    void *out;
    long long qs[3], os[3];
    const int *lengths, *q_lengths;
    int parts, kv_heads, group, q_len, kv_len, hd;
    int window, right, sinks;
    int out_dtype;
    float scale_log2;
};

template <int D, int NT> struct TokensShape {
    static constexpr int BLOCK = CacheBlock<D>::BYTES;
    static constexpr int STAGES = 6;
    static constexpr int RING = kWarps * STAGES * BLOCK;
    static constexpr int ROWS = 8 * NT;
    // The parts' place at the end, over the ring: m, l of the warps and the CTA, outputs.
    static constexpr int PARTS = (2 * kWarps + 2) * ROWS * 4 + kWarps * ROWS * (D + 4) * 4;
    static constexpr int SMEM = RING > PARTS ? RING : PARTS;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <int N> __device__ __forceinline__ void shared_words(uint32_t at, uint32_t *w) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}
__device__ __forceinline__ void copy_async_16(uint32_t to, const uint8_t *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(const void *p, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ float peer_load(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// Which columns lane c holds: words of 8 columns.  Its words lie together where a token's
// row is a power of two of bytes; at 96 columns (48 bytes) it takes every fourth word, which
// meets all banks.
template <int D> struct Columns {
    static constexpr bool TOGETHER = D != 96;
    static constexpr int WORDS = D / 32;
    __device__ static constexpr int first(int word, int c) { return TOGETHER ? c * (D / 4) + word * 8 : word * 32 + c * 8; }
};

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : 2) window_e2m1_tokens_kernel(const __grid_constant__ TokensParams p) {
    using S = TokensShape<D, NT>;
    using B = CacheBlock<D>;
    using C = Columns<D>;
    constexpr int ROWS = S::ROWS, ST = S::STAGES;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int parts = p.parts, pair = blockIdx.x / parts, part = blockIdx.x - pair * parts;
    const int b = pair / p.kv_heads, kvh = pair - b * p.kv_heads;
    const int n = max(0, min(p.lengths[b], p.kv_len));
    const int m = p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
    const int row0 = blockIdx.y * ROWS, rows = min(ROWS, p.group * m - row0);
    // Rows r of the tile: query (row0 + r) / group, head kvh * group + (row0 + r) % group.
    const int pos0 = n - m;

    // Keys that some row of the tile sees: [0, sink) and [low, high); blocks [0, sink_blocks)
    // and from `begin` on.
    const int first = pos0 + row0 / p.group, last = pos0 + (row0 + max(rows, 1) - 1) / p.group;
    const int high = rows > 0 ? max(0, min(n, last + p.right + 1)) : 0;
    const int low = p.window > 0 ? max(0, min(first - p.window + 1, high)) : 0;
    const int sink = min(p.sinks, low);
    const int sink_blocks = (sink + kCacheBlock - 1) / kCacheBlock;
    const int begin = max(low / kCacheBlock, sink_blocks);
    const int blocks = sink_blocks + max(0, (high + kCacheBlock - 1) / kCacheBlock - begin);
    const int stride = parts * kWarps;
    const int limit_all = min(n, first + p.right + 1), floor_all = p.window > 0 ? last - p.window + 1 : 0;

    // The queries as B operands, and the masks of columns 2c and 2c + 1.
    uint32_t qb[NT][D / 16][2];
    float factor[NT][2]; // from S to log2 units
    int limit[NT][2], floor_[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 8 * t + g;
        const bool real = 8 * t + g < rows;
        const uint16_t *q = p.q + b * p.qs[0] + (kvh * p.group + r % p.group) * p.qs[1] + (r / p.group) * p.qs[2];
        uint4 w[C::WORDS];
        uint32_t top2 = 0;
#pragma unroll
        for (int j = 0; j < C::WORDS; ++j) {
            const int col = C::first(j, c);
            w[j] = real && col < p.hd ? *reinterpret_cast<const uint4 *>(q + col) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t *x = &w[j].x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                top2 = __vmaxu2(top2, x[e] & 0x7fff7fffu);
        }
        int exponent = 0; // q is multiplied by 2^exponent
        if constexpr (BF16) {
            uint32_t top = max(top2 & 0xffffu, top2 >> 16);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // The largest element is in [2^(e - 127), 2^(e - 126)); a row that is not finite stays as it is.
            const int e = static_cast<int>(top >> 7);
            exponent = e == 255 ? 0 : min(141 - e, 120);
            const float times = __uint_as_float(static_cast<uint32_t>(exponent + 127) << 23);
#pragma unroll
            for (int j = 0; j < C::WORDS; ++j) {
                uint32_t *x = &w[j].x;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[i] = pack_f16(__uint_as_float(x[i] << 16) * times, __uint_as_float(x[i] & 0xffff0000u) * times);
            }
        }
#pragma unroll
        for (int j = 0; j < C::WORDS; ++j) {
            qb[t][2 * j][0] = w[j].x;
            qb[t][2 * j][1] = w[j].y;
            qb[t][2 * j + 1][0] = w[j].z;
            qb[t][2 * j + 1][1] = w[j].w;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int col = 8 * t + 2 * c + h, pos = pos0 + (row0 + col) / p.group;
            const int of_col = __shfl_sync(0xffffffffu, exponent, 4 * (2 * c + h));
            factor[t][h] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - of_col) << 23);
            limit[t][h] = col < rows ? min(n, pos + p.right + 1) : n; // a row that is none: anything finite
            floor_[t][h] = col < rows && p.window > 0 ? pos - p.window + 1 : 0;
        }
    }

    float o[NT][D / 16][4];
    float ref[NT][2], sum[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
            o[t][x][0] = o[t][x][1] = o[t][x][2] = o[t][x][3] = 0.f;
        ref[t][0] = ref[t][1] = -INFINITY;
        sum[t][0] = sum[t][1] = 0.f;
    }

    auto block_of = [&](int i) { return i < sink_blocks ? i : begin + i - sink_blocks; };
    const uint32_t ring = smem_u32(smem) + warp * ST * S::BLOCK;
    uint32_t missing = 0; // bit per stage: its page is none of the cache's
    auto fetch = [&](int i, int stage) {
        int within;
        const int page = p.cache.page_of(b, block_of(i), within);
        missing = page < 0 ? missing | 1u << stage : missing & ~(1u << stage);
        if (page < 0)
            return;
        const uint8_t *from = p.cache.block_at(page, kvh, within, S::BLOCK);
        const uint32_t to = ring + stage * S::BLOCK;
#pragma unroll
        for (int x = lane * 16; x < S::BLOCK; x += 512)
            copy_async_16(to + x, from + x);
    };
    int i = part * kWarps + warp;
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) {
        if (i + k * stride < blocks)
            fetch(i + k * stride, k);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int stage = 0; i < blocks; i += stride, stage = stage + 1 == ST ? 0 : stage + 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
        __syncwarp(); // this block has landed for every lane, and every lane is done with the last one
        const bool bad = missing >> stage & 1u;
        if (i + (ST - 1) * stride < blocks)
            fetch(i + (ST - 1) * stride, stage == 0 ? ST - 1 : stage - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t at = ring + stage * S::BLOCK;

        // S^T: tokens g (rows 0 to 7) and g + 8.
        uint32_t kw[2][C::WORDS], scales[C::TOGETHER ? 1 : C::WORDS];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t row = at + B::KEYS + (g + 8 * h) * (D / 2);
            if constexpr (C::TOGETHER)
                shared_words<C::WORDS>(row + c * 4 * C::WORDS, kw[h]);
            else
#pragma unroll
                for (int j = 0; j < C::WORDS; ++j)
                    shared_words<1>(row + j * 16 + c * 4, &kw[h][j]);
        }
#pragma unroll
        for (int j = 0; j < (C::TOGETHER ? 1 : C::WORDS); ++j) // both tokens' scales of the lane's group
            shared_words<1>(at + B::KEY_SCALES + 2 * B::key_scale(g, C::first(j, c) / 32), &scales[j]);
        float s[NT][4], s2[NT][4]; // two chains of dependent products
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[t][e] = s2[t][e] = 0.f;
#pragma unroll
        for (int j = 0; j < C::WORDS; ++j) {
            const uint32_t both = scales[C::TOGETHER ? 0 : j];
            const uint32_t s_g = __byte_perm(both, 0, 0x1010), s_g8 = __byte_perm(both, 0, 0x3232);
            uint32_t x[4], y[4];
            f16x8(kw[0][j], x);
            f16x8(kw[1][j], y);
            const uint32_t a0[4] = {hmul2(x[0], s_g), hmul2(y[0], s_g8), hmul2(x[1], s_g), hmul2(y[1], s_g8)};
            const uint32_t a1[4] = {hmul2(x[2], s_g), hmul2(y[2], s_g8), hmul2(x[3], s_g), hmul2(y[3], s_g8)};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma16816(s[t], a0, qb[t][2 * j][0], qb[t][2 * j][1]);
                mma16816(s2[t], a1, qb[t][2 * j + 1][0], qb[t][2 * j + 1][1]);
            }
        }
        const int key = block_of(i) * kCacheBlock;
        // A block that every row sees whole needs no mask.
        const bool whole = !bad && key + kCacheBlock <= limit_all && (key >= floor_all || key + kCacheBlock <= p.sinks);
        bool above = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) { // token g + 8 (e / 2), query 2c + e % 2
                float x = (s[t][e] + s2[t][e]) * factor[t][e & 1];
                if (!whole) {
                    const int token = key + g + 8 * (e >> 1);
                    const bool seen = token < limit[t][e & 1] && (token >= floor_[t][e & 1] || token < p.sinks);
                    x = seen ? (bad ? NAN : x) : -INFINITY;
                }
                s[t][e] = x;
                above |= x > ref[t][e & 1] + kLazy;
            }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float times[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float top = fmaxf(s[t][h], s[t][h + 2]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = fmaxf(top, ref[t][h]);
                    times[h] = top > ref[t][h] ? ex2_approx(ref[t][h] - top) : 1.f;
                    ref[t][h] = top;
                    sum[t][h] *= times[h];
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    o[t][x][0] *= times[0];
                    o[t][x][1] *= times[1];
                    o[t][x][2] *= times[0];
                    o[t][x][3] *= times[1];
                }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float r = ref[t][e & 1];
                s[t][e] = ex2_approx(s[t][e] - (r == -INFINITY ? 0.f : r));
                sum[t][e & 1] += s[t][e];
            }
            pb[t][0] = turn(pack_f16(s[t][0], s[t][1]));
            pb[t][1] = turn(pack_f16(s[t][2], s[t][3]));
        }

        // O^T: a lane's scales are those of tokens 2c, 2c + 1 and 2c + 8, 2c + 9.
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (!whole) { // values that no row sees may be anything: their scale is zero
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                keep[h] = 0;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int token = key + 2 * c + 8 * h + e;
                    if (!bad && token < high && (token >= low || token < sink))
                        keep[h] |= 0xffffu << (16 * e);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < D / 16 / B::W; ++v) {
            uint32_t vw[B::W];
            shared_words<B::W>(at + B::VALUES + B::value_word(v * B::W, lane), vw);
#pragma unroll
            for (int j = 0; j < B::W; j += 2) {
                uint32_t vs[2]; // one group of 32 columns
                shared_words<2>(at + B::VALUE_SCALES + 2 * B::value_scale(2 * c, (v * B::W + j) / 2), vs);
                vs[0] &= keep[0];
                vs[1] &= keep[1];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t x[4];
                    f16x8(vw[j + e], x);
                    const uint32_t a[4] = {hmul2(x[0], vs[0]), hmul2(x[1], vs[0]), hmul2(x[2], vs[1]), hmul2(x[3], vs[1])};
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        mma16816(o[t][v * B::W + j + e], a, pb[t][0], pb[t][1]);
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads(); // the ring becomes the parts' place
    float(*part_m)[ROWS] = reinterpret_cast<float(*)[ROWS]>(smem), (*part_l)[ROWS] = part_m + kWarps;
    float *cta_m = part_l[kWarps], *cta_l = cta_m + ROWS;
    float(*part_o)[ROWS][D + 4] = reinterpret_cast<float(*)[ROWS][D + 4]>(cta_l + ROWS);

    // The warps' parts, then the CTAs': out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 4);
            sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 8);
            sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 16);
            const int r = 8 * t + 2 * c + h;
            if (g == 0) {
                part_m[warp][r] = ref[t][h];
                part_l[warp][r] = sum[t][h];
            }
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                part_o[warp][r][16 * x + g] = o[t][x][h];
                part_o[warp][r][16 * x + 8 + g] = o[t][x][2 + h];
            }
        }
    __syncthreads();
    for (int x = threadIdx.x; x < ROWS * D; x += kWarps * 32) {
        const int r = x / D, col = x - r * D;
        float mx = part_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w)
            mx = fmaxf(mx, part_m[w][r]);
        const float base = mx == -INFINITY ? 0.f : mx;
        float l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(part_m[w][r] - base);
            l += f * part_l[w][r];
            v += f * part_o[w][r][col];
        }
        part_o[0][r][col] = v;
        if (col == 0) {
            cta_m[r] = mx;
            cta_l[r] = l;
        }
    }
    if (parts > 1)
        cluster_sync();
    else
        __syncthreads();
    for (int x = part * kWarps * 32 + threadIdx.x; x < ROWS * D; x += parts * kWarps * 32) {
        const int r = x / D, col = x - r * D;
        if (r >= rows || col >= p.hd)
            continue;
        float l, v;
        if (parts > 1) {
            float mx = -INFINITY;
            for (int k = 0; k < parts; ++k)
                mx = fmaxf(mx, peer_load(peer(&cta_m[r], k)));
            const float base = mx == -INFINITY ? 0.f : mx;
            l = v = 0.f;
            for (int k = 0; k < parts; ++k) {
                const float f = exp2f(peer_load(peer(&cta_m[r], k)) - base);
                l += f * peer_load(peer(&cta_l[r], k));
                v += f * peer_load(peer(&part_o[0][r][col], k));
            }
        } else {
            l = cta_l[r];
            v = part_o[0][r][col];
        }
        const int row = row0 + r;
        // Zeros for a row that sees no key, which its position tells: a sum that is no
        // positive number otherwise stands for scores that are not finite, and gives NaN.
        v = min(n, pos0 + row / p.group + p.right + 1) > 0 ? v / l : 0.f;
        const long long to = b * p.os[0] + (kvh * p.group + row % p.group) * p.os[1] + (row / p.group) * p.os[2] + col;
        if (p.out_dtype == kOutF32)
            static_cast<float *>(p.out)[to] = v;
        else if (p.out_dtype == kOutBF16)
            static_cast<__nv_bfloat16 *>(p.out)[to] = __float2bfloat16_rn(v);
        else
            static_cast<__half *>(p.out)[to] = __float2half_rn(v);
    }
    if (parts > 1)
        cluster_sync(); // no CTA leaves while another reads its part
}

template <int D, int NT, bool BF16> int launch_rows(const TokensParams &p, int batch, cudaStream_t stream) {
    using S = TokensShape<D, NT>;
    static std::atomic<unsigned long long> done{0};
    const void *kernel = reinterpret_cast<const void *>(window_e2m1_tokens_kernel<D, NT, BF16>);
    const cudaError_t e = set_smem_limit(kernel, S::SMEM, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    if (p.parts > 8) { // clusters above 8 CTAs need the kernel's consent
        const cudaError_t w = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (w != cudaSuccess)
            return static_cast<int>(w);
    }
    const int tiles = (p.group * p.q_len + S::ROWS - 1) / S::ROWS;
    cudaLaunchConfig_t cfg{};
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.gridDim = dim3(static_cast<unsigned>(p.parts) * batch * p.kv_heads, tiles);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, window_e2m1_tokens_kernel<D, NT, BF16>, p));
}
template <int D> int launch_d(const TokensParams &p, int batch, bool bf16, cudaStream_t stream) {
    if (p.group * p.q_len <= 8)
        return bf16 ? launch_rows<D, 1, true>(p, batch, stream) : launch_rows<D, 1, false>(p, batch, stream);
    return bf16 ? launch_rows<D, 2, true>(p, batch, stream) : launch_rows<D, 2, false>(p, batch, stream);
}

} // namespace

// CTAs that split the keys of one tile of rows: until four (two of 16 rows) are on every SM,
// with two blocks left for each warp.
int window_e2m1_tokens_parts(const WindowE2m1Args &a) {
    const long long rows = static_cast<long long>(a.heads / a.cache.kv_heads) * a.cache.q_len;
    const long long tile = rows <= 8 ? 8 : 16, tiles = (rows + tile - 1) / tile;
    const long long ctas = tiles * a.cache.batch * a.cache.kv_heads, most = (rows <= 8 ? 4ll : 2ll) * fmha_sm_count();
    long long keys = a.kv_len;
    if (a.window > 0)
        keys = std::min(keys, static_cast<long long>(a.window) + a.cache.q_len + a.right + a.sinks);
    int parts = 1;
    while (parts < kMaxParts && ctas * parts * 2 <= most && keys >= 2ll * parts * 2 * kWarps * kCacheBlock)
        parts *= 2;
    return parts;
}

int window_e2m1_tokens_launch(const WindowE2m1Args &a, cudaStream_t stream) {
    TokensParams p{};
    const CacheArgs &c = a.cache;
    p.cache.data = static_cast<uint8_t *>(c.data);
    p.cache.table = c.table;
    p.cache.page_stride = c.page_stride;
    p.cache.head_stride = c.head_stride;
    p.cache.pages = c.pages;
    p.cache.page_blocks = c.page_tokens / kCacheBlock;
    p.cache.table_width = c.table_width;
    p.q = static_cast<const uint16_t *>(a.q);
    p.out = a.out;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a.qs[i];
        p.os[i] = a.os[i];
    }
    p.lengths = c.lengths;
    p.q_lengths = c.q_lengths;
    p.kv_heads = c.kv_heads;
    p.group = a.heads / c.kv_heads;
    p.q_len = c.q_len;
    p.kv_len = a.kv_len;
    p.hd = c.hd;
    p.window = a.window;
    p.right = a.right;
    p.sinks = a.sinks;
    p.out_dtype = a.out_dtype;
    const double scale = a.scale > 0 ? a.scale : 1.0 / std::sqrt(static_cast<double>(c.hd));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.parts = window_e2m1_tokens_parts(a);
    const bool bf16 = a.dtype == kBF16;
    switch (cache_width(c.hd)) {
    case 32:
        return launch_d<32>(p, c.batch, bf16, stream);
    case 64:
        return launch_d<64>(p, c.batch, bf16, stream);
    case 96:
        return launch_d<96>(p, c.batch, bf16, stream);
    default:
        return launch_d<128>(p, c.batch, bf16, stream);
    }
}

// A workspace means: the keys and values go back to 16 bits there (exactly), and the
// prompts' kernel reads them.
size_t window_e2m1_workspace(const WindowE2m1Args &a) {
    const CacheArgs &c = a.cache;
    const long long rows = static_cast<long long>(a.heads / c.kv_heads) * c.q_len, tiles = (rows + 15) / 16;
    if (tiles <= 4)
        return 0;
    return 4ull * c.batch * c.kv_heads * a.kv_len * c.hd;
}

int window_e2m1_launch(const WindowE2m1Args &a, cudaStream_t stream) {
    const size_t bytes = window_e2m1_workspace(a);
    if (bytes == 0)
        return window_e2m1_tokens_launch(a, stream);
    const CacheArgs &c = a.cache;
    WindowArgs w;
    w.q = a.q;
    w.k = a.workspace;
    w.v = static_cast<uint8_t *>(a.workspace) + bytes / 2;
    w.out = a.out;
    w.batch = c.batch;
    w.heads = a.heads;
    w.kv_heads = c.kv_heads;
    w.q_len = c.q_len;
    w.kv_len = a.kv_len;
    w.hd = c.hd;
    const long long strides[3] = {static_cast<long long>(c.kv_heads) * a.kv_len * c.hd,
                                  static_cast<long long>(a.kv_len) * c.hd, c.hd};
    for (int i = 0; i < 3; ++i) {
        w.qs[i] = a.qs[i];
        w.os[i] = a.os[i];
        w.ks[i] = w.vs[i] = strides[i];
    }
    w.lengths = c.lengths;
    w.q_lengths = c.q_lengths;
    w.window = a.window;
    w.right = a.right;
    w.sinks = a.sinks;
    w.bf16 = a.dtype == kBF16;
    w.out_dtype = a.out_dtype;
    w.scale = a.scale;
    w.err = a.err;
    CacheReadRange range;
    range.whole = true;
    range.kv_len = a.kv_len;
    range.window = a.window;
    range.sinks = a.sinks;
    const int rc = cache_read_launch(c, const_cast<void *>(w.k), const_cast<void *>(w.v), strides, strides, a.dtype, range, stream);
    return rc ? rc : window_prompt_launch(w, stream);
}

} // namespace omni_b200
