// linear_e4m3_sm100.cu -- matrix product in 8-bit floating point with block
// scales, for B200 (sm_100a).
//
//   out[m, n] = sum_g sa[m, g] * sw[n / 128, g] * (sum_{k in group g} a[m, k] w[n, k]) + bias[n]
//
// a and w are e4m3, a group is 128 columns of k, the scales are fp32.  The
// inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4, fp32
// accumulators in TMEM), one group at a time: a scale belongs to one group, so
// each group's 128-column product is read back from TMEM, multiplied by its
// two scales and added to fp32 sums in registers.  Two TMEM accumulators let
// the tensor cores run one group ahead.
#include "e4m3.cuh"
#include "layer.h"
#include "sm100.cuh"
#include "tma.h"

#include <algorithm>

namespace omni_b200 {
namespace {

struct LinearParams {
    CUtensorMap ta, tw, to;
    const float *sa, *sw;
    const void *bias;
    void *out;
    long long ldo;
    int m, n, groups;
    int m_tiles, n_tiles;
    int out_dtype, o_tma;
    int *err;
};

constexpr int kRowBytes = 128; // a tile row: one group of e4m3

template <int N> __device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Bounded by time only: nothing may be in flight when the CTA gives back its
// shared memory and TMEM.
__device__ __forceinline__ void drain_wait(uint64_t *bar, uint32_t parity, int *err) {
    const uint32_t a = smem_u32(bar);
    const uint64_t start = globaltimer_ns();
    while (!mbar_try_wait(a, parity)) {
        if (globaltimer_ns() - start > kWaitLimitNs) {
            atomicOr(err, kErrWaitDrain);
            return;
        }
    }
}

__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int *err, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

// Two fp32 sums in one 64-bit register pair.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
// sum += d * s.  volatile: the sums of one TMEM load are taken before the next
// load's registers are filled.
__device__ __forceinline__ void add_scaled(uint64_t &sum, uint32_t d0, uint32_t d1, uint64_t s) {
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\tfma.rn.f32x2 %0, d, %3, %0;\n\t}"
                 : "+l"(sum)
                 : "r"(d0), "r"(d1), "l"(s));
}

__device__ __forceinline__ float bias_at(const LinearParams &p, int n) {
    if (!p.bias || n >= p.n)
        return 0.f;
    if (p.out_dtype == kF32)
        return static_cast<const float *>(p.bias)[n];
    if (p.out_dtype == kBF16)
        return __bfloat162float(static_cast<const __nv_bfloat16 *>(p.bias)[n]);
    return __half2float(static_cast<const __half *>(p.bias)[n]);
}
__device__ __forceinline__ void store_one(const LinearParams &p, long long at, float v) {
    if (p.out_dtype == kF32)
        static_cast<float *>(p.out)[at] = v;
    else if (p.out_dtype == kBF16)
        static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p.out)[at] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dtype) {
    if (dtype == kBF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// ------------------------------------------------------------ large products
// Persistent CTAs, tiles of 128 rows x 256 columns of out.  Warps 0-7 add up:
// warp w owns TMEM lane quarter w % 4 (32 rows, a row per lane) and columns
// [128 (w / 4), +128), which lie in one block of w, so a thread's 128 sums all
// take the same factor.  Warp 8 loads, warp 9 issues the products.  Registers:
// 384 x 168 at launch = 256 x 224 (sums) + 128 x 56 (control).
constexpr int kBigM = 128, kBigN = 256, kBigStages = 4, kBigThreads = 384;
constexpr int kBigStageBytes = (kBigM + kBigN) * kRowBytes;
constexpr int kStagingBytes = 8 * 32 * 128; // a 32-row x 128-byte output box per warp
constexpr int kBigSmem = kBigStages * kBigStageBytes + kStagingBytes + 256 + 1024;
constexpr int kBand = 16; // row tiles of a band

// Tile order: bands of 16 row tiles, rows first, so that the tiles that run
// together span few rows of a and of w.
__device__ __forceinline__ void tile_at(const LinearParams &p, int tile, int &mt, int &nt) {
    const int per_band = kBand * p.n_tiles;
    const int band = tile / per_band, in = tile - band * per_band;
    const int rows = min(kBand, p.m_tiles - band * kBand);
    nt = in / rows;
    mt = band * kBand + in - nt * rows;
}

__global__ void __launch_bounds__(kBigThreads, 1) linear_e4m3_big(const __grid_constant__ LinearParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t *staging = smem + kBigStages * kBigStageBytes;
    uint64_t *full = reinterpret_cast<uint64_t *>(staging + kStagingBytes);
    uint64_t *empty = full + kBigStages;
    uint64_t *acc_full = empty + kBigStages; // [2]
    uint64_t *acc_empty = acc_full + 2;      // [2]
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = p.m_tiles * p.n_tiles;
    int *err = p.err;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kBigStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8);
        }
        mbar_init(drain, 1);
        fence_mbarrier_init();
    }
    if (warp == 9) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp >= 8) {
        reg_dec<56>();
        if (warp == 8) {
            int n = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                int mt, nt;
                tile_at(p, tile, mt, nt);
                for (int g = 0; g < p.groups; ++g, ++n) {
                    const int st = n % kBigStages;
                    if (!(ok = warp_wait(&empty[st], ((n / kBigStages) & 1) ^ 1, err, kErrWaitEmpty)))
                        break;
                    if (elect_one()) {
                        uint8_t *to = smem + st * kBigStageBytes;
                        mbar_arrive_expect_tx(&full[st], kBigStageBytes);
                        tma_load_2d(to, &p.ta, &full[st], g * kRowBytes, mt * kBigM);
                        tma_load_2d(to + kBigM * kRowBytes, &p.tw, &full[st], g * kRowBytes, nt * kBigN);
                    }
                    __syncwarp();
                }
            }
            for (int j = max(0, n - kBigStages); j < n; ++j)
                drain_wait(&full[j % kBigStages], (j / kBigStages) & 1, err);
        } else if (warp == 9) {
            constexpr uint32_t idesc = make_idesc_e4m3(kBigM, kBigN);
            const uint32_t leader = elect_one() ? 1u : 0u;
            const uint32_t base = smem_u32(smem);
            int n = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                for (int g = 0; g < p.groups; ++g, ++n) {
                    const int st = n % kBigStages, buf = n & 1;
                    if (!(ok = warp_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, err, kErrWaitAcc)))
                        break;
                    if (!(ok = warp_wait(&full[st], (n / kBigStages) & 1, err, kErrWaitK)))
                        break;
                    tc_fence_after();
                    const uint32_t at = base + st * kBigStageBytes;
                    const uint64_t ad = make_smem_desc(at, 16, 8 * kRowBytes, kLayoutSW128);
                    const uint64_t wd = make_smem_desc(at + kBigM * kRowBytes, 16, 8 * kRowBytes, kLayoutSW128);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_ss_f8_if(leader, tmem + buf * kBigN, ad + 2 * k, wd + 2 * k, idesc, k > 0 ? 1u : 0u);
                    tc_commit_if(leader, &empty[st]);
                    tc_commit_if(leader, &acc_full[buf]);
                    __syncwarp();
                }
            }
            tc_commit_if(leader, drain);
            drain_wait(drain, 0, err);
        }
        __syncwarp();
    } else {
        reg_inc<224>();
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
        uint8_t *box = staging + warp * 4096;
        int n = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
            int mt, nt;
            tile_at(p, tile, mt, nt);
            const int row = mt * kBigM + quarter * 32 + lane;
            const int col = nt * kBigN + half * 128;
            // Rows and blocks past the end have scale 0 (their operands are zero fill).
            const bool real = row < p.m && col < p.n;
            const float *sa = p.sa + static_cast<long long>(real ? row : 0) * p.groups;
            const float *sw = p.sw + static_cast<long long>(real ? col / 128 : 0) * p.groups;
            uint64_t acc[64]; // 128 sums, starting at the bias
#pragma unroll
            for (int c = 0; c < 64; ++c)
                acc[c] = pair(bias_at(p, col + 2 * c), bias_at(p, col + 2 * c + 1));
            float a_next = __ldg(sa), w_next = __ldg(sw);
            for (int g = 0; g < p.groups; ++g, ++n) {
                const float f = a_next * w_next;
                const uint64_t s = pair(f, f);
                if (g + 1 < p.groups) {
                    a_next = __ldg(sa + g + 1);
                    w_next = __ldg(sw + g + 1);
                }
                const int buf = n & 1;
                if (!(ok = warp_wait(&acc_full[buf], (n >> 1) & 1, err, kErrWaitS)))
                    break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t d[32];
                    tmem_ld32(lanes + buf * kBigN + c, d);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        add_scaled(acc[(c + e) / 2], d[e], d[e + 1], s);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&acc_empty[buf]);
            }
            if (!ok)
                break;
            // A box of 32 rows x 128 bytes at a time, each lane its row, in the
            // 128-byte swizzle of the store's tensor map; rows that TMA cannot
            // address leave the box by plain stores.
            const int r0 = mt * kBigM + quarter * 32;
            auto reuse = [&]() {
                if (lane == 0)
                    tma_store_wait_read();
                __syncwarp();
            };
            auto flush = [&](int c, int size) {
                fence_proxy_async_smem();
                __syncwarp();
                if (r0 >= p.m || c >= p.n)
                    return;
                if (p.o_tma) {
                    if (lane == 0) {
                        tma_store_2d(&p.to, box, c, r0);
                        tma_store_commit();
                    }
                    return;
                }
                const int width = min(128 / size, p.n - c);
                for (int r = 0; r < 32 && r0 + r < p.m; ++r)
                    for (int j = lane; j < width; j += 32) {
                        const uint8_t *from = box + r * 128 + ((((j * size) >> 4) ^ (r & 7)) << 4) + ((j * size) & 15);
                        const long long at = (r0 + r) * p.ldo + c + j;
                        if (size == 4)
                            static_cast<uint32_t *>(p.out)[at] = *reinterpret_cast<const uint32_t *>(from);
                        else
                            static_cast<uint16_t *>(p.out)[at] = *reinterpret_cast<const uint16_t *>(from);
                    }
                __syncwarp();
            };
            if (p.out_dtype == kF32) {
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    reuse();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 v0 = unpair(acc[c / 2 + j * 2]), v1 = unpair(acc[c / 2 + j * 2 + 1]);
                        *reinterpret_cast<float4 *>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                            make_float4(v0.x, v0.y, v1.x, v1.y);
                    }
                    flush(col + c, 4);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 128; c += 64) {
                    reuse();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 v = unpair(acc[c / 2 + j * 4 + e]);
                            w[e] = pack16(v.x, v.y, p.out_dtype);
                        }
                        *reinterpret_cast<uint4 *>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    flush(col + c, 2);
                }
            }
        }
        if (lane == 0)
            tma_store_wait_read();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9)
        tmem_dealloc(tmem, 512);
}

// --------------------------------------------------------------- few rows
// The tensor cores take 128 rows of w as their 128 lanes and T rows of a as
// columns, so a call with few rows reads each block of w once and wastes no
// lanes.  A cluster of `gridDim.x` CTAs splits the groups of one (128 x T) tile
// of out, so that enough SMs load w; each leaves its sums in shared memory and
// the cluster adds them in rank order (no atomics: the same result each time).
// Warps 0-3: sums, lane quarter = warp; 4 loads; 5 issues the products.
template <int T> struct FewShape {
    static constexpr int STAGE = 128 * kRowBytes + T * kRowBytes;
    static constexpr int STAGES = 180 * 1024 / STAGE;
    static constexpr int SUMS = T * 128 * 4; // over the ring, when every product is done
    static constexpr int SCALES = 2 * T * 4;
    static constexpr int SMEM = STAGES * STAGE + SCALES + 512 + 1024;
    static constexpr int TMEM = 2 * T < 32 ? 32 : 2 * T;
    static_assert(SUMS <= STAGES * STAGE, "the sums fit in the ring");
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_load(uint32_t addr, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <int T> __global__ void __launch_bounds__(192, 1) linear_e4m3_few(const __grid_constant__ LinearParams p) {
    using S = FewShape<T>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float *scales = reinterpret_cast<float *>(smem + S::STAGES * S::STAGE); // [2][T]
    uint64_t *full = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(scales) + S::SCALES);
    uint64_t *empty = full + S::STAGES;
    uint64_t *acc_full = empty + S::STAGES;
    uint64_t *acc_empty = acc_full + 2;
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
    static_assert((2 * S::STAGES + 6) * 8 <= 512, "barrier space");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = gridDim.x, part = blockIdx.x;
    const int g0 = part * p.groups / parts, g1 = (part + 1) * p.groups / parts;
    const int n0 = blockIdx.y * 128, m0 = blockIdx.z * T;
    int *err = p.err;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 4);
        }
        mbar_init(drain, 1);
        fence_mbarrier_init();
    }
    if (warp == 5) {
        tmem_alloc(tmem_holder, S::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    float acc[T];
    if (warp == 4) {
        bool ok = true;
        int n = 0;
        for (int g = g0; ok && g < g1; ++g, ++n) {
            const int st = n % S::STAGES;
            if (!(ok = warp_wait(&empty[st], ((n / S::STAGES) & 1) ^ 1, err, kErrWaitEmpty)))
                break;
            if (elect_one()) {
                uint8_t *to = smem + st * S::STAGE;
                mbar_arrive_expect_tx(&full[st], S::STAGE);
                tma_load_2d(to, &p.tw, &full[st], g * kRowBytes, n0);
                tma_load_2d(to + 128 * kRowBytes, &p.ta, &full[st], g * kRowBytes, m0);
            }
            __syncwarp();
        }
        for (int j = max(0, n - S::STAGES); j < n; ++j)
            drain_wait(&full[j % S::STAGES], (j / S::STAGES) & 1, err);
        __syncwarp();
    } else if (warp == 5) {
        constexpr uint32_t idesc = make_idesc_e4m3(128, T);
        const uint32_t leader = elect_one() ? 1u : 0u;
        const uint32_t base = smem_u32(smem);
        bool ok = true;
        int n = 0;
        for (int g = g0; ok && g < g1; ++g, ++n) {
            const int st = n % S::STAGES, buf = n & 1;
            if (!(ok = warp_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, err, kErrWaitAcc)))
                break;
            if (!(ok = warp_wait(&full[st], (n / S::STAGES) & 1, err, kErrWaitK)))
                break;
            tc_fence_after();
            const uint32_t at = base + st * S::STAGE;
            const uint64_t wd = make_smem_desc(at, 16, 8 * kRowBytes, kLayoutSW128);
            const uint64_t ad = make_smem_desc(at + 128 * kRowBytes, 16, 8 * kRowBytes, kLayoutSW128);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                umma_ss_f8_if(leader, tmem + buf * T, wd + 2 * k, ad + 2 * k, idesc, k > 0 ? 1u : 0u);
            tc_commit_if(leader, &empty[st]);
            tc_commit_if(leader, &acc_full[buf]);
            __syncwarp();
        }
        tc_commit_if(leader, drain);
        drain_wait(drain, 0, err);
        __syncwarp();
    } else {
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
#pragma unroll
        for (int j = 0; j < T; ++j)
            acc[j] = 0.f;
        // Thread j < T fetches the scale of a's row m0 + j one group ahead.
        const int t = threadIdx.x;
        const bool mine = t < T && m0 + t < p.m;
        const float *sa = p.sa + static_cast<long long>(mine ? m0 + t : 0) * p.groups;
        const float *sw = p.sw + static_cast<long long>(n0 / 128) * p.groups;
        float a_next = mine && g0 < g1 ? __ldg(sa + g0) : 0.f, w_next = g0 < g1 ? __ldg(sw + g0) : 0.f;
        bool ok = true;
        int n = 0;
        for (int g = g0; g < g1; ++g, ++n) {
            const int buf = n & 1;
            if (t < T)
                scales[buf * T + t] = a_next * w_next;
            if (g + 1 < g1) {
                a_next = mine ? __ldg(sa + g + 1) : 0.f;
                w_next = __ldg(sw + g + 1);
            }
            // The scales of this group are written, those of the last but one read.
            asm volatile("bar.sync 1, 128;" ::: "memory");
            ok = ok && warp_wait(&acc_full[buf], (n >> 1) & 1, err, kErrWaitS);
            if (!ok)
                continue; // the other warps of bar 1 count on this one
            tc_fence_after();
            const float4 *f = reinterpret_cast<const float4 *>(scales + buf * T);
            constexpr int C = T < 32 ? 16 : 32;
#pragma unroll
            for (int c = 0; c < T; c += C) {
                uint32_t d[C];
                if constexpr (C == 32)
                    tmem_ld32(lanes + buf * T + c, d);
                else
                    tmem_ld16(lanes + buf * T + c, d);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < C; e += 4) {
                    const float4 s = f[(c + e) / 4];
                    ffma2(acc[c + e], acc[c + e + 1], __uint_as_float(d[e]), __uint_as_float(d[e + 1]), s.x, s.y,
                          acc[c + e], acc[c + e + 1]);
                    ffma2(acc[c + e + 2], acc[c + e + 3], __uint_as_float(d[e + 2]), __uint_as_float(d[e + 3]), s.z,
                          s.w, acc[c + e + 2], acc[c + e + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&acc_empty[buf]);
        }
    }
    // Every copy has landed and every product is done before the ring becomes
    // the sums' place.
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 5)
        tmem_dealloc(tmem, S::TMEM);
    const int col = n0 + static_cast<int>(threadIdx.x);
    const bool writes = threadIdx.x < 128 && col < p.n;
    if (parts == 1) {
        if (writes) {
            const float b = bias_at(p, col);
#pragma unroll
            for (int j = 0; j < T; ++j)
                if (m0 + j < p.m)
                    store_one(p, (m0 + j) * p.ldo + col, acc[j] + b);
        }
        return;
    }
    float *sums = reinterpret_cast<float *>(smem); // [T][128]
    if (threadIdx.x < 128) {
#pragma unroll
        for (int j = 0; j < T; ++j)
            sums[j * 128 + threadIdx.x] = acc[j];
    }
    cluster_sync();
    if (writes) {
        const float b = bias_at(p, col);
        for (int j = part; j < T && m0 + j < p.m; j += parts) {
            const uint32_t at = smem_u32(sums + j * 128 + threadIdx.x);
            float v = 0.f;
            for (int r = 0; r < parts; ++r)
                v += peer_load(at, r);
            store_one(p, (m0 + j) * p.ldo + col, v + b);
        }
    }
    cluster_sync(); // no CTA leaves while another reads its sums
}

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
        n = 148;
    return n;
}

template <int T> int launch_few(LinearParams &p, const LinearArgs &a, int parts, cudaStream_t stream) {
    using S = FewShape<T>;
    int rc = 0;
    if ((rc = make_map_pitched(&p.ta, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, a.m, a.lda, kRowBytes, T)) ||
        (rc = make_map_pitched(&p.tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, a.n, a.ldw, kRowBytes, 128)))
        return rc;
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(linear_e4m3_few<T>), S::SMEM, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(parts, (a.n + 127) / 128, (a.m + T - 1) / T);
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, linear_e4m3_few<T>, p));
}

int launch_big(LinearParams &p, const LinearArgs &a, int sms, cudaStream_t stream) {
    int rc = 0;
    if ((rc = make_map_pitched(&p.ta, a.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, a.m, a.lda, kRowBytes, kBigM)) ||
        (rc = make_map_pitched(&p.tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.k, a.n, a.ldw, kRowBytes, kBigN)))
        return rc;
    const int size = a.out_dtype == kF32 ? 4 : 2;
    p.o_tma = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ldo * size % 16 == 0;
    if (p.o_tma) {
        const CUtensorMapDataType type = a.out_dtype == kF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : a.out_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        if ((rc = make_map_pitched(&p.to, a.out, type, size, a.n, a.m, a.ldo * size, 128 / size, 32)))
            return rc;
    }
    p.m_tiles = (a.m + kBigM - 1) / kBigM;
    p.n_tiles = (a.n + kBigN - 1) / kBigN;
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(linear_e4m3_big), kBigSmem, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
    linear_e4m3_big<<<static_cast<unsigned>(std::min<long long>(tiles, sms)), kBigThreads, kBigSmem, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

} // namespace

int linear_e4m3_launch(const LinearArgs &a, cudaStream_t stream) {
    LinearParams p{};
    p.sa = a.a_scales;
    p.sw = a.w_scales;
    p.bias = a.bias;
    p.out = a.out;
    p.ldo = a.ldo;
    p.m = a.m;
    p.n = a.n;
    p.groups = (a.k + kGroup - 1) / kGroup;
    p.out_dtype = a.out_dtype;
    p.err = a.err;
    const int sms = sm_count();
    const long long big = static_cast<long long>((a.m + kBigM - 1) / kBigM) * ((a.n + kBigN - 1) / kBigN);
    if (a.m > 128 && 2 * big >= sms)
        return launch_big(p, a, sms, stream);
    // Split the groups over up to 8 CTAs while the tiles leave SMs idle.
    const int t = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
    const long long tiles = static_cast<long long>((a.n + 127) / 128) * ((a.m + t - 1) / t);
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= sms && parts * 2 <= p.groups)
        parts *= 2;
    switch (t) {
    case 16:
        return launch_few<16>(p, a, parts, stream);
    case 32:
        return launch_few<32>(p, a, parts, stream);
    case 64:
        return launch_few<64>(p, a, parts, stream);
    default:
        return launch_few<128>(p, a, parts, stream);
    }
}

} // namespace omni_b200
