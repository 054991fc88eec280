// window_tokens.cu -- sliding-window attention for few queries: the next tokens
// of sequences against their caches.
//
// softmax(scale * q k^T + mask) v for the `group * q_len` query rows that share
// a key head, 16 of them at a time as the rows of mma.sync m16n8k16.  Every key
// and value that a row may see is read once per 16 rows, so the bound is the
// memory traffic of the caches.  (A 128-row tcgen05 tile would be 15/16 empty;
// here the tensor work stays far below the loads.)
//
// Keys go to the warps 16 at a time; each warp keeps its own running maximum,
// sum and output and copies its keys and values to a ring of its own in shared
// memory (cp.async, two chunks ahead, no barrier between warps).  The fragments
// leave it by 16-byte loads, by a choice of index order:
//   q k^T sums over the head dimension in any order: in each 32 columns, lane
//     quad index c = lane % 4 holds columns 8c..8c+7 of q and of k, and takes
//     them as the k-indexes (2c, 2c+1, 2c+8, 2c+9) of two mma steps;
//   p v gives its columns in any order: column index n = lane / 4 of mma j
//     stands for column 8n + j (of each 64), so lane / 4 loads columns 8n..8n+7
//     of its four keys and pairs them up with byte permutes.
// Rows are 128 or 256 bytes apart; the 16-byte pieces of a row are permuted by
// the row number so that the eight lanes of a load phase meet all 32 banks.
// 64 sequences of up to 16384 keys, 32/8 heads of 128, window 4096: 167 us, 6.19 TB/s.
// A cluster of CTAs splits the keys of one tile of rows, so that few sequences
// still load with many SMs; the parts meet in distributed shared memory, in rank
// order (no atomics).
#include "fmha.h"
#include "sm100.cuh"

#include <algorithm>
#include <cmath>

namespace omni_b200 {
namespace {

constexpr int kWarps = 4, kChunk = 16, kStages = 3, kMaxParts = 16;

struct TokensParams {
    const uint16_t *q, *k, *v;
    void *out;
    long long qs[3], ks[3], vs[3], os[3];
    const int *lengths, *q_lengths;
    int parts, kv_heads, group, q_len, kv_len, hd;
    int window, right, sinks;
    int out_dtype;
    float scale_log2;
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint4 load16(const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// 16 bytes to shared memory, zeros where `real` is false (nothing is read then).
__device__ __forceinline__ void copy_async_16(uint32_t to, const uint16_t *from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
// Low and high halves of two words: (x.lo, y.lo) and (x.hi, y.hi).
__device__ __forceinline__ uint32_t lows(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x5410); }
__device__ __forceinline__ uint32_t highs(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x7632); }

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

template <int DK> struct TokensShape {
    static constexpr int DV = (DK + 1) / 2;         // 64-column steps of v
    static constexpr int PITCH = DV * 128;          // bytes of a row
    static constexpr int TILE = kChunk * PITCH;     // a chunk's keys, or values
    static constexpr int RING = kWarps * kStages * 2 * TILE;
    static constexpr int D = DK * 32;
    // The parts' place at the end, over the ring: m, l of the warps and the CTA, outputs.
    static constexpr int PARTS = (2 * kWarps + 2) * 16 * 4 + kWarps * 16 * (D + 4) * 4;
    static constexpr int SMEM = RING > PARTS ? RING : PARTS;
};

// DK: 32-column steps of the head dimension; columns past hd are zeros.
template <int DK, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 2) window_tokens_kernel(const __grid_constant__ TokensParams p) {
    using S = TokensShape<DK>;
    constexpr int DV = S::DV, D = S::D;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int parts = p.parts, pair = blockIdx.x / parts, part = blockIdx.x - pair * parts;
    const int b = pair / p.kv_heads, kvh = pair - b * p.kv_heads;
    const int n = p.lengths ? max(0, min(p.lengths[b], p.kv_len)) : p.kv_len;
    const int m = p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
    const int row0 = blockIdx.y * 16, rows = min(16, p.group * m - row0);
    // Rows r of the tile: query (row0 + r) / group, head kvh * group + (row0 + r) % group.
    const int pos0 = n - m;
    const uint16_t *kb = p.k + b * p.ks[0] + kvh * p.ks[1], *vb = p.v + b * p.vs[0] + kvh * p.vs[1];

    // Keys that some row of the tile sees: [0, sink) and [low, high).
    const int first = pos0 + row0 / p.group, last = pos0 + (row0 + max(rows, 1) - 1) / p.group;
    const int high = rows > 0 ? max(0, min(n, last + p.right + 1)) : 0;
    const int low = p.window > 0 ? max(0, min(first - p.window + 1, high)) : 0;
    const int sink = min(p.sinks, low);
    const int sink_chunks = (sink + kChunk - 1) / kChunk;
    const int chunks = sink_chunks + (high - low + kChunk - 1) / kChunk;
    const int stride = parts * kWarps;

    // This thread's rows g and g + 8: their keys [.., limit) with [sinks, floor) hidden.
    int limit[2], floor_[2];
    const int limit_all = min(n, first + p.right + 1), floor_all = p.window > 0 ? last - p.window + 1 : 0;
    uint32_t qa[DK * 2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = row0 + g + 8 * h;
        const bool real = g + 8 * h < rows;
        const int pos = pos0 + r / p.group;
        limit[h] = real ? min(n, pos + p.right + 1) : n; // a row that is none: anything finite
        floor_[h] = real && p.window > 0 ? pos - p.window + 1 : 0;
        const uint16_t *q = p.q + b * p.qs[0] + (kvh * p.group + r % p.group) * p.qs[1] + (r / p.group) * p.qs[2];
#pragma unroll
        for (int d = 0; d < DK; ++d) {
            const int col = d * 32 + c * 8;
            const uint4 w = real && col < p.hd ? load16(q + col) : make_uint4(0u, 0u, 0u, 0u);
            qa[2 * d][h] = w.x;
            qa[2 * d][2 + h] = w.y;
            qa[2 * d + 1][h] = w.z;
            qa[2 * d + 1][2 + h] = w.w;
        }
    }
    float o[DV * 8][4];
#pragma unroll
    for (int j = 0; j < DV * 8; ++j)
        o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    // First key and end of chunk i.
    auto chunk_at = [&](int i, int &key, int &end) {
        key = i < sink_chunks ? i * kChunk : low + (i - sink_chunks) * kChunk;
        end = i < sink_chunks ? sink : high;
    };
    const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * S::TILE;
    auto fetch = [&](int i, int stage) {
        int key, end;
        chunk_at(i, key, end);
        const uint32_t to = ring + stage * 2 * S::TILE;
        constexpr int P = DK * 4; // pieces of a row
#pragma unroll
        for (int x = lane; x < kChunk * P; x += 32) {
            const int row = x / P, j = x - row * P;
            const bool real = key + row < end && j * 8 < p.hd;
            const long long s = real ? key + row : 0;
            const int at = real ? j * 8 : 0;
            const uint32_t piece = row * S::PITCH + (j & ~7) * 16;
            copy_async_16(to + piece + (((j & 7) ^ ((row & 1) << 2 | ((row >> 1) & 3))) << 4), kb + s * p.ks[2] + at, real);
            copy_async_16(to + S::TILE + piece + (((j & 7) ^ (row & 7)) << 4), vb + s * p.vs[2] + at, real);
        }
    };
    int i = part * kWarps + warp;
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) {
        if (i + k * stride < chunks)
            fetch(i + k * stride, k);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int stage = 0; i < chunks; i += stride, stage = stage + 1 == kStages ? 0 : stage + 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp(); // this chunk has landed for every lane, and every lane is done with the last one
        if (i + (kStages - 1) * stride < chunks)
            fetch(i + (kStages - 1) * stride, stage == 0 ? kStages - 1 : stage - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const uint32_t kt = ring + stage * 2 * S::TILE, vt = kt + S::TILE;
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float s2[4] = {0.f, 0.f, 0.f, 0.f}; // a second chain of dependent products
            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
            const uint32_t row = kt + (t * 8 + g) * S::PITCH, turn = (g & 1) << 2 | ((g >> 1) & 3);
#pragma unroll
            for (int d = 0; d < DK; ++d) {
                const int j = d * 4 + c;
                const uint4 k = shared16(row + (j & ~7) * 16 + (((j & 7) ^ turn) << 4));
                mma16816<BF16>(s[t], qa[2 * d], k.x, k.y);
                mma16816<BF16>(s2, qa[2 * d + 1], k.z, k.w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[t][e] += s2[e];
        }
        int key, end;
        chunk_at(i, key, end);
        // A chunk that every row sees whole needs no mask.
        const bool whole = key + kChunk <= min(end, limit_all) && (key >= floor_all || key + kChunk <= p.sinks);
        // s[t][2h + e]: row g + 8h, key + 8t + 2c + e.
        float grown[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int at = key + t * 8 + c * 2 + e;
                    float &x = s[t][2 * h + e];
                    const bool seen = whole || (at < end && at < limit[h] && (at >= floor_[h] || at < p.sinks));
                    x = seen ? x * p.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(mx, top[h]);
            grown[h] = mx > top[h] ? ex2_approx(top[h] - mx) : 1.f;
            top[h] = mx;
            const float ref = mx == -INFINITY ? 0.f : mx;
            sum[h] *= grown[h];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float &x = s[t][2 * h + e];
                    x = ex2_approx(x - ref);
                    sum[h] += x;
                }
        }
        if (__any_sync(0xffffffffu, grown[0] != 1.f || grown[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < DV * 8; ++j) {
                o[j][0] *= grown[0];
                o[j][1] *= grown[0];
                o[j][2] *= grown[1];
                o[j][3] *= grown[1];
            }
        }
        // The tensor cores multiply 16-bit operands: P loses up to half a step of its type
        // here (the sums above are of the unrounded values).  One sequence's next token in
        // bf16 is off by 0.0019 (root mean square, relative) where fp32 weights give 0.0016,
        // the rounding of the output alone; products in fp32 would leave the tensor cores.
        const uint32_t pa[4] = {pack_pair<BF16>(s[0][0], s[0][1]), pack_pair<BF16>(s[0][2], s[0][3]),
                                pack_pair<BF16>(s[1][0], s[1][1]), pack_pair<BF16>(s[1][2], s[1][3])};
#pragma unroll
        for (int d = 0; d < DV; ++d) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = c * 2 + (e & 1) + (e >> 1) * 8;
                v[e] = shared16(vt + row * S::PITCH + d * 128 + ((g ^ (row & 7)) << 4));
            }
            const uint32_t *x0 = &v[0].x, *x1 = &v[1].x, *x2 = &v[2].x, *x3 = &v[3].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mma16816<BF16>(o[d * 8 + 2 * j], pa, lows(x0[j], x1[j]), lows(x2[j], x3[j]));
                mma16816<BF16>(o[d * 8 + 2 * j + 1], pa, highs(x0[j], x1[j]), highs(x2[j], x3[j]));
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads(); // the ring becomes the parts' place
    float(*part_m)[16] = reinterpret_cast<float(*)[16]>(smem), (*part_l)[16] = part_m + kWarps;
    float *cta_m = part_l[kWarps], *cta_l = cta_m + 16;
    float(*part_o)[16][D + 4] = reinterpret_cast<float(*)[16][D + 4]>(cta_l + 16);

    // The warps' parts, then the CTAs': out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        if (c == 0) {
            part_m[warp][g + 8 * h] = top[h];
            part_l[warp][g + 8 * h] = sum[h];
        }
#pragma unroll
        for (int j = 0; j < DV * 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // Column index 2c + e of mma j of 64-column step j / 8.
                const int col = (j / 8) * 64 + (2 * c + e) * 8 + (j & 7);
                if (col < D)
                    part_o[warp][g + 8 * h][col] = o[j][2 * h + e];
            }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * D; x += kWarps * 32) {
        const int r = x / D, col = x - r * D;
        float mx = part_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w)
            mx = fmaxf(mx, part_m[w][r]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float l = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2f(part_m[w][r] - ref);
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
    for (int x = part * kWarps * 32 + threadIdx.x; x < 16 * D; x += parts * kWarps * 32) {
        const int r = x / D, col = x - r * D;
        if (r >= rows || col >= p.hd)
            continue;
        float l, v;
        if (parts > 1) {
            float mx = -INFINITY;
            for (int k = 0; k < parts; ++k)
                mx = fmaxf(mx, peer_load(peer(&cta_m[r], k)));
            const float ref = mx == -INFINITY ? 0.f : mx;
            l = v = 0.f;
            for (int k = 0; k < parts; ++k) {
                const float f = exp2f(peer_load(peer(&cta_m[r], k)) - ref);
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
        const long long at = b * p.os[0] + (kvh * p.group + row % p.group) * p.os[1] + (row / p.group) * p.os[2] + col;
        if (p.out_dtype == kOutF32)
            static_cast<float *>(p.out)[at] = v;
        else if (p.out_dtype == kOutBF16)
            static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
        else
            static_cast<__half *>(p.out)[at] = __float2half_rn(v);
    }
    if (parts > 1)
        cluster_sync(); // no CTA leaves while another reads its part
}

template <int DK, bool BF16> int launch_dk(const TokensParams &p, dim3 grid, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(window_tokens_kernel<DK, BF16>),
                                         TokensShape<DK>::SMEM, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    if (p.parts > 8) { // clusters above 8 CTAs need the kernel's consent
        const cudaError_t w = cudaFuncSetAttribute(window_tokens_kernel<DK, BF16>,
                                                   cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (w != cudaSuccess)
            return static_cast<int>(w);
    }
    cudaLaunchConfig_t cfg{};
    cfg.dynamicSmemBytes = TokensShape<DK>::SMEM;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = p.parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, window_tokens_kernel<DK, BF16>, p));
}

template <bool BF16> int launch_type(const TokensParams &p, dim3 grid, cudaStream_t stream) {
    switch ((p.hd + 31) / 32) {
    case 1:
        return launch_dk<1, BF16>(p, grid, stream);
    case 2:
        return launch_dk<2, BF16>(p, grid, stream);
    case 3:
        return launch_dk<3, BF16>(p, grid, stream);
    default:
        return launch_dk<4, BF16>(p, grid, stream);
    }
}

} // namespace

// CTAs that split the keys of one tile of rows: until two are on every SM, with two
// chunks left for each warp.  Measured, 4101 keys x 128: 512 tiles 168 us with one
// part, 180 with two; 128 tiles 36 and 28 us (four: 30); 32 tiles 38 us with two
// parts, 23 with four, 20 with eight.
int window_tokens_parts(const WindowArgs &a) {
    const long long tiles = (static_cast<long long>(a.heads / a.kv_heads) * a.q_len + 15) / 16;
    const long long ctas = tiles * a.batch * a.kv_heads, most = 2ll * fmha_sm_count();
    long long keys = a.kv_len;
    if (a.window > 0)
        keys = std::min(keys, static_cast<long long>(a.window) + a.q_len + a.right + a.sinks);
    int parts = 1;
    while (parts < kMaxParts && ctas * parts * 2 <= most && keys >= 2ll * parts * 2 * kWarps * kChunk)
        parts *= 2;
    return parts;
}

int window_tokens_launch(const WindowArgs &a, cudaStream_t stream) {
    TokensParams p{};
    p.q = static_cast<const uint16_t *>(a.q);
    p.k = static_cast<const uint16_t *>(a.k);
    p.v = static_cast<const uint16_t *>(a.v);
    p.out = a.out;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a.qs[i];
        p.ks[i] = a.ks[i];
        p.vs[i] = a.vs[i];
        p.os[i] = a.os[i];
    }
    p.lengths = a.lengths;
    p.q_lengths = a.q_lengths;
    p.kv_heads = a.kv_heads;
    p.group = a.heads / a.kv_heads;
    p.q_len = a.q_len;
    p.kv_len = a.kv_len;
    p.hd = a.hd;
    p.window = a.window;
    p.right = a.right;
    p.sinks = a.sinks;
    p.out_dtype = a.out_dtype;
    const double scale = a.scale > 0 ? a.scale : 1.0 / std::sqrt(static_cast<double>(a.hd));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    const int parts = window_tokens_parts(a), tiles = (p.group * a.q_len + 15) / 16;
    p.parts = parts;
    const dim3 grid(static_cast<unsigned>(parts) * a.batch * a.kv_heads, tiles);
    return a.bf16 ? launch_type<true>(p, grid, stream) : launch_type<false>(p, grid, stream);
}

} // namespace omni_b200
