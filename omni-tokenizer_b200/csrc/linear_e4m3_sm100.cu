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
// That way out of TMEM, once a group, is the bound of large products: 8192 x 8192 x
// 4096 251 us (2186 TFLOP/s; the tensor pipe is 54 % busy, TMEM's 60 %), 24000 x 4096 x
// 1024 with bias 122 us.  Few rows read w once: 1 x 4096 x 4096 6 us.
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
// sum += d * f.  volatile: the sums of one TMEM load are taken before a later
// load's registers are filled.
__device__ __forceinline__ void add_scaled(uint64_t &sum, uint32_t d0, uint32_t d1, uint64_t f) {
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\tfma.rn.f32x2 %0, d, %3, %0;\n\t}"
                 : "+l"(sum)
                 : "r"(d0), "r"(d1), "l"(f));
}
__device__ __forceinline__ float shared_f32(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 shared_f32x4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
// Arrives without release: for a thread whose reads so far are complete (their
// values are in registers) and that has written nothing.  The release form would
// wait for every load in flight.
__device__ __forceinline__ void arrive_relaxed(uint64_t *bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.relaxed.cta.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(bar))
                 : "memory");
}
// 4 bytes from global to shared memory, asynchronously.
__device__ __forceinline__ void copy_async_4(float *dst, const float *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrives on `bar` when this thread's copies so far have landed.
__device__ __forceinline__ void copy_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 16 bytes to shared memory by a 32-bit address: the sums leave few registers.
__device__ __forceinline__ void put16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
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
// A box's elements to rows r0.. and columns col.. of out, one warp.
__device__ __forceinline__ void store_box(const LinearParams &p, const uint8_t *box, int r0, int col, int size) {
    const int width = min(128 / size, p.n - col), rows = min(32, p.m - r0);
    for (int r = 0; r < rows; ++r)
        for (int j = lane_id(); j < width; j += 32) {
            const int at = j * size;
            const uint8_t *from = box + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15);
            const long long to = (r0 + r) * p.ldo + col + j;
            if (size == 4)
                static_cast<uint32_t *>(p.out)[to] = *reinterpret_cast<const uint32_t *>(from);
            else
                static_cast<uint16_t *>(p.out)[to] = *reinterpret_cast<const uint16_t *>(from);
        }
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
// take the same factor.  Warp 8 loads, warps 9 and 10 issue the products.  Registers:
// 384 x 168 at launch = 256 x 216 (sums) + 128 x 72 (control).
constexpr int kBigM = 128, kBigN = 256, kBigStages = 3, kBigThreads = 384;
constexpr int kSumWarps = 8, kLoadWarp = 8, kIssueWarp = 9;
constexpr int kBigStageBytes = (kBigM + kBigN) * kRowBytes;
// Two output boxes of 32 rows x 128 bytes per warp: all of a warp's 2-byte
// outputs, so that a tile waits for no store of its own.
constexpr int kBoxBytes = 32 * 128;
// The scales of a group: 128 of a's rows and two of w's blocks.  Loading stage n
// of the ring follows product n - 3, which follows the sums of group n - 5, so
// eight slots need no barrier of their own.
constexpr int kScaleSlots = 8, kSlotFloats = kBigM + 4;
static_assert(kScaleSlots >= kBigStages + 2, "a slot is read before it is written again");
constexpr int kBigSmem =
    kBigStages * kBigStageBytes + kSumWarps * 2 * kBoxBytes + kScaleSlots * kSlotFloats * 4 +
    kSumWarps * 512 + 256 + 1024;
static_assert(kBigSmem <= 227 * 1024, "shared memory of a CTA");
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
    float *scales = reinterpret_cast<float *>(staging + kSumWarps * 2 * kBoxBytes);
    float *bias_lines = scales + kScaleSlots * kSlotFloats; // [warp][128]
    uint64_t *full = reinterpret_cast<uint64_t *>(bias_lines + kSumWarps * 128);
    // Product n is done: its accumulator is full, and its stage n % 3 free.
    uint64_t *done = full + kBigStages;
    uint64_t *acc_empty = done + kBigStages; // [2]
    uint64_t *drain = acc_empty + 2;         // [2]
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = p.m_tiles * p.n_tiles;
    int *err = p.err;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kBigStages; ++s) {
            mbar_init(&full[s], 33); // 32 lanes' copies of the scales, and the tensor copies' bytes
            mbar_init(&done[s], 2);  // the product's end, and its issuer, which saw the scales
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_empty[i], kSumWarps);
            mbar_init(&drain[i], 1);
        }
        fence_mbarrier_init();
    }
    if (warp == kIssueWarp) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp >= kLoadWarp) {
        reg_dec<72>();
        if (warp == kLoadWarp) {
            int n = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                int mt, nt;
                tile_at(p, tile, mt, nt);
                // Rows and columns past the end: their operands are zero fill.
                const float *sa[4], *sw = p.sw + static_cast<long long>(min(nt * 2 + (lane & 1), (p.n - 1) / 128)) * p.groups;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sa[i] = p.sa + static_cast<long long>(min(mt * kBigM + i * 32 + lane, p.m - 1)) * p.groups;
                for (int g = 0; g < p.groups; ++g, ++n) {
                    const int st = n % kBigStages;
                    if (!(ok = warp_wait(&done[st], ((n / kBigStages) & 1) ^ 1, err, kErrWaitEmpty)))
                        break;
                    if (elect_one()) {
                        uint8_t *to = smem + st * kBigStageBytes;
                        mbar_arrive_expect_tx(&full[st], kBigStageBytes);
                        tma_load_2d(to, &p.ta, &full[st], g * kRowBytes, mt * kBigM);
                        tma_load_2d(to + kBigM * kRowBytes, &p.tw, &full[st], g * kRowBytes, nt * kBigN);
                    }
                    float *slot = scales + (n % kScaleSlots) * kSlotFloats;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        copy_async_4(slot + i * 32 + lane, sa[i] + g);
                    if (lane < 2)
                        copy_async_4(slot + kBigM + lane, sw + g);
                    copy_async_arrive(&full[st]);
                    __syncwarp();
                }
            }
            for (int j = max(0, n - kBigStages); j < n; ++j)
                drain_wait(&full[j % kBigStages], (j / kBigStages) & 1, err);
        } else if (warp < kIssueWarp + 2) {
            // One warp alone cannot issue as fast as the products run (its waits
            // and commits cost it about 600 clocks a group, a product 512), so
            // each of two owns an accumulator and takes every other group.
            constexpr uint32_t idesc = make_idesc_e4m3(kBigM, kBigN);
            const uint32_t leader = elect_one() ? 1u : 0u;
            const uint32_t base = smem_u32(smem);
            const int buf = warp - kIssueWarp;
            int total = 0;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x)
                total += p.groups;
            for (int n = buf; n < total; n += 2) {
                const int st = n % kBigStages;
                if (!warp_wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1, err, kErrWaitAcc) ||
                    !warp_wait(&full[st], (n / kBigStages) & 1, err, kErrWaitK))
                    break;
                tc_fence_after();
                const uint32_t at = base + st * kBigStageBytes;
                const uint64_t ad = make_smem_desc(at, 16, 8 * kRowBytes, kLayoutSW128);
                const uint64_t wd = make_smem_desc(at + kBigM * kRowBytes, 16, 8 * kRowBytes, kLayoutSW128);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_ss_f8_if(leader, tmem + buf * kBigN, ad + 2 * k, wd + 2 * k, idesc, k > 0 ? 1u : 0u);
                tc_commit_if(leader, &done[st]);
                if (leader)
                    mbar_arrive(&done[st]);
                __syncwarp();
            }
            tc_commit_if(leader, &drain[buf]);
            drain_wait(&drain[buf], 0, err);
        }
        __syncwarp();
    } else {
        reg_inc<216>();
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
        const uint32_t box = smem_u32(staging) + warp * 2 * kBoxBytes;
        const uint32_t biases = smem_u32(bias_lines);
        const uint32_t own_scale = smem_u32(scales) + (quarter * 32 + lane) * 4, block_scale = smem_u32(scales) + (kBigM + half) * 4;
        int n = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
            int mt, nt;
            tile_at(p, tile, mt, nt);
            const int r0 = mt * kBigM + quarter * 32;
            const int col = nt * kBigN + half * 128;
            // Bias of columns col + 4 lane.., wanted when the sums are complete.
            float bias[4] = {0.f, 0.f, 0.f, 0.f};
            if (p.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    bias[e] = bias_at(p, col + 4 * lane + e);
            }
            uint64_t acc[64]; // 128 sums
#pragma unroll
            for (int c = 0; c < 64; ++c)
                acc[c] = 0;
            for (int g = 0; g < p.groups; ++g, ++n) {
                const int buf = n & 1;
                if (!(ok = warp_wait(&done[n % kBigStages], (n / kBigStages) & 1, err, kErrWaitS)))
                    break;
                tc_fence_after();
                const uint32_t slot = (n % kScaleSlots) * (kSlotFloats * 4);
                const float s = shared_f32(own_scale + slot) * shared_f32(block_scale + slot);
                const uint64_t f = pair(s, s);
#pragma unroll
                for (int c = 0; c < 128; c += 16) {
                    uint32_t d[16];
                    tmem_ld16(lanes + buf * kBigN + c, d);
                    tmem_wait_ld();
                    if (c == 112) { // all of it is in registers: the next product may start
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0)
                            arrive_relaxed(&acc_empty[buf]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        add_scaled(acc[(c + e) / 2], d[e], d[e + 1], f);
                }
            }
            if (!ok)
                break;
            // Boxes of 32 rows x 128 bytes, each lane its row, in the 128-byte swizzle
            // of the store's tensor map; rows that TMA cannot address leave the box
            // by plain stores.
            const int size = p.out_dtype == kF32 ? 4 : 2, width = 128 / size;
            const uint32_t line = biases + warp * 512; // the bias in column order
            if (p.bias) {
                __syncwarp();
                put16(line + lane * 16, __float_as_uint(bias[0]), __float_as_uint(bias[1]), __float_as_uint(bias[2]),
                      __float_as_uint(bias[3]));
            }
#pragma unroll
            for (int c = 0; c < 128; c += 16) {
                // 16 columns: half a box of fp32, a quarter of one of 2-byte elements.
                const int in = c % width, which = (c / width) & 1;
                if (size == 4 ? c % 64 == 0 : c == 0) { // both boxes are free again
                    if (lane == 0)
                        tma_store_wait_read();
                    __syncwarp();
                }
                float v[16];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 x = unpair(acc[c / 2 + e]);
                    v[2 * e] = x.x;
                    v[2 * e + 1] = x.y;
                }
                if (p.bias) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 b = shared_f32x4(line + (c + e) * 4);
                        v[e] += b.x;
                        v[e + 1] += b.y;
                        v[e + 2] += b.z;
                        v[e + 3] += b.w;
                    }
                }
                const uint32_t row = box + which * kBoxBytes + lane * 128;
                auto place = [&](int j) { return row + ((j ^ (lane & 7)) << 4); };
                if (size == 4) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        put16(place(j + in / 4), __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                              __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        put16(place(j + in / 8), pack16(v[8 * j], v[8 * j + 1], p.out_dtype),
                              pack16(v[8 * j + 2], v[8 * j + 3], p.out_dtype),
                              pack16(v[8 * j + 4], v[8 * j + 5], p.out_dtype),
                              pack16(v[8 * j + 6], v[8 * j + 7], p.out_dtype));
                }
                if (in + 16 < width)
                    continue;
                const int at = col + c + 16 - width; // the box's first column
                fence_proxy_async_smem();
                __syncwarp();
                if (r0 >= p.m || at >= p.n)
                    continue;
                uint8_t *from = staging + (warp * 2 + which) * kBoxBytes;
                if (p.o_tma) {
                    if (lane == 0) {
                        tma_store_2d(&p.to, from, at, r0);
                        tma_store_commit();
                    }
                } else {
                    store_box(p, from, r0, at, size);
                    __syncwarp();
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
    if (warp == kIssueWarp)
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
        // Eight rows at a time: their loads from a peer are in flight together.
        for (int j0 = part; j0 < T && m0 + j0 < p.m; j0 += 8 * parts) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = b;
            for (int r = 0; r < parts; ++r) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = peer_load(smem_u32(sums + min(j0 + i * parts, T - 1) * 128 + threadIdx.x), r);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] += x[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = j0 + i * parts;
                if (j < T && m0 + j < p.m)
                    store_one(p, (m0 + j) * p.ldo + col, v[i]);
            }
        }
    }
    cluster_sync(); // no CTA leaves while another reads its sums
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
    const int sms = fmha_sm_count();
    // Few rows: the groups are split over up to 8 CTAs while the tiles leave SMs idle.
    // Clusters of four and eight do not reach the last SMs of a GPC: 128 at once.
    const int t = a.m <= 16 ? 16 : a.m <= 32 ? 32 : a.m <= 64 ? 64 : 128;
    const long long tiles = static_cast<long long>((a.n + 127) / 128) * ((a.m + t - 1) / t);
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= (parts >= 2 ? std::min(sms, 128) : sms) && parts * 2 <= p.groups)
        parts *= 2;
    // The cheaper kernel, in tenths of a microsecond as measured (launch, then groups
    // one after another): 4096 x 4096, few rows / large tiles: m 1 6.1 / 17.1 us, m 64
    // 9.8 / 17.6, m 128 13.7 / 18.2, m 256 20.3 / 18.1; 8192 x 1024: m 33 7.8 / 8.1, m
    // 128 13.1 / 8.6; 1152 x 4304: m 384 13.9 / 24.9.
    const long long big = static_cast<long long>((a.m + kBigM - 1) / kBigM) * ((a.n + kBigN - 1) / kBigN);
    const long long at_once = parts >= 4 ? std::min(sms, 128) : sms;
    const long long few_cost =
        50 + t / 4 + (tiles * parts + at_once - 1) / at_once * ((p.groups + parts - 1) / parts) * (2 + t / 25);
    const long long big_cost = 50 + (big + sms - 1) / sms * p.groups * 4;
    if (big_cost < few_cost)
        return launch_big(p, a, sms, stream);
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
