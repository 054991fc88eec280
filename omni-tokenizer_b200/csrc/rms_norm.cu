// rms_norm.cu -- root-mean-square norm with the residual's addition, and the
// quantisation to e4m3 with a scale for each 128 columns (rows) or each 128 x
// 128 block (weights).
//
// Per row, in fp32 (inputs are widened, the sum is not rounded before the norm
// reads it):
//   h = x + residual,  y = h * rsqrt(mean(h^2) + eps) * weight,
// residual_out = h and out = y, each rounded once to the element type, or out =
// the groups of e4m3.cuh.  A row is read once: its elements stay in registers
// between the sum of squares and the scaling (vector kernel), so the bound is
// the memory traffic of the inputs and outputs: 16384 x 8192 bf16 with a residual to
// e4m3 148 us, 6.37 TB/s; 24000 x 4096 bf16 to e4m3 49 us, 6.0 TB/s.
//
// quantize_rows_kernel: rows to e4m3 without a norm.
// rows_kernel: TPR threads own a row, 8 consecutive elements each per step
// (16-byte loads of 2-byte types), VPT steps.  A group of 128 columns is then
// 16 neighbouring lanes, so its largest magnitude takes four shuffles and no
// shared memory.  The grid is persistent: the weight is read once per CTA.
// rows_stream_kernel: many rows.  The same thread layout, rows through a ring of
// shared memory that bulk copies fill several rows ahead, so that loads are in
// flight at all times.
// rows_odd_kernel serves columns and pitches that 16-byte loads cannot,
// rows_scalar_kernel rows wider than the registers hold; it reads its row twice (the
// second time from L2).  Both move an element a load, and write e4m3 a byte a store, so
// that instructions bound them, not the traffic: 17679 x 3727 bf16 with a residual to
// e4m3 129 us, 3.6 TB/s, with the issue slots 67 % busy and DRAM 40 %.
#include "e4m3.cuh"
#include "layer.h"
#include "sm100.cuh"

#include <algorithm>

namespace omni_b200 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Over the 16 lanes of a half warp.
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1)
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// Thread t's elements of a row to `out`, as they are or in groups of e4m3.
template <typename T, bool QUANT, int TPR, int VPT>
__device__ __forceinline__ void write_row(const RowsArgs &a, long long row, int groups, int t, float (&h)[VPT][8]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * TPR + t) * 8;
        if constexpr (QUANT) {
            const float scale = group_scale(half_warp_max(amax8(h[i])));
            if (c < a.cols) {
                uint8_t *q = static_cast<uint8_t *>(a.out) + row * a.out_stride + c;
                *reinterpret_cast<uint2 *>(q) = e4m3x8<false>(h[i], divisor_of(scale));
                if (t % 16 == 0)
                    a.scales[row * groups + c / kGroup] = scale;
            }
        } else if (c < a.cols) {
            store8(static_cast<T *>(a.out) + row * a.out_stride + c, pack8<T>(h[i]));
        }
    }
}

template <typename T, bool QUANT, int TPR, int VPT, int ROWS>
__global__ void __launch_bounds__(TPR *ROWS) rows_kernel(const RowsArgs a) {
    constexpr int WARPS = TPR / 32; // warps of a row
    __shared__ float part[2][WARPS];
    static_assert(ROWS == 1 || TPR == 32, "a row of one warp, or a CTA for each row");
    const int t = threadIdx.x % TPR;
    const T *x = static_cast<const T *>(a.x), *res = static_cast<const T *>(a.residual);
    T *res_out = static_cast<T *>(a.residual_out);
    const int groups = (a.cols + kGroup - 1) / kGroup;
    Vec8<T> w[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * TPR + t) * 8;
        if (c < a.cols)
            w[i] = load8(static_cast<const T *>(a.weight) + c);
    }
    int turn = 0;
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    // The next row's loads are under way while this one is reduced, scaled and written
    // (23328 x 1152: 47 -> 38 us).
    Vec8<T> xv[VPT], rv[VPT];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < a.cols) {
                xv[i] = load8(x + row * a.x_stride + c);
                if (res)
                    rv[i] = load8(res + row * a.residual_stride + c);
            }
        }
    };
    long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / TPR;
    if (row < a.rows)
        fetch(row);
    for (; row < a.rows; row += step) {
        float h[VPT][8];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < a.cols) {
                unpack8(xv[i], h[i]);
                if (res) {
                    float r[8];
                    unpack8(rv[i], r);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        h[i][e] += r[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    h[i][e] = 0.f;
            }
        }
        if (row + step < a.rows)
            fetch(row + step);
        if (res) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * TPR + t) * 8;
                if (c < a.cols)
                    store8(res_out + row * a.residual_out_stride + c, pack8<T>(h[i]));
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sum = fmaf(h[i][e], h[i][e], sum);
        sum = warp_sum(sum);
        if constexpr (WARPS > 1) {
            // Two buffers: a warp may write the next row's part while
            // another still reads this row's.
            if (t % 32 == 0)
                part[turn][t / 32] = sum;
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k)
                sum += part[turn][k];
            turn ^= 1;
        }
        const float rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < a.cols) {
                float wf[8];
                unpack8(w[i], wf);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    h[i][e] = h[i][e] * rstd * wf[e];
            }
        }
        write_row<T, QUANT, TPR, VPT>(a, row, groups, t, h);
    }
}

constexpr int kStreamThreads = 256, kStreamBytes = 96 * 1024, kMaxStages = 8;

__device__ __forceinline__ void bulk_load(uint32_t to, const void *from, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                 "l"(from), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// 256 / TPR rows at a time.  Stage: their x, then their residuals, `pitch` bytes
// each.  Elements go to registers at once, so a stage is filled again while the
// row is reduced, scaled and written.
template <typename T, bool QUANT, int TPR, int VPT>
__global__ void __launch_bounds__(kStreamThreads) rows_stream_kernel(const RowsArgs a, int stages) {
    constexpr int ROWS = kStreamThreads / TPR, WARPS = TPR / 32;
    static_assert(WARPS > 1, "narrow rows are rows_kernel's");
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kMaxStages];
    __shared__ float part[2][kStreamThreads / 32];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const bool res = a.residual != nullptr;
    const uint32_t pitch = a.cols * sizeof(T), stage_bytes = ROWS * pitch * (res ? 2 : 1);
    const int groups = (a.cols + kGroup - 1) / kGroup;
    const long long turns = (a.rows + ROWS - 1) / ROWS;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i)
            mbar_init(&full[i], 1);
        fence_mbarrier_init();
    }
    __syncthreads();
    // Rows [turn * ROWS, ..) into a stage (thread 0).
    int filled = 0;
    auto fill = [&](long long turn, int stage) {
        ++filled;
        const long long row = turn * ROWS;
        const int rows = static_cast<int>(min(static_cast<long long>(ROWS), a.rows - row));
        const uint32_t to = smem_u32(ring) + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], rows * pitch * (res ? 2 : 1));
        for (int r = 0; r < rows; ++r) {
            bulk_load(to + r * pitch, static_cast<const T *>(a.x) + (row + r) * a.x_stride, pitch, &full[stage]);
            if (res)
                bulk_load(to + (ROWS + r) * pitch, static_cast<const T *>(a.residual) + (row + r) * a.residual_stride,
                          pitch, &full[stage]);
        }
    };
    if (threadIdx.x == 0)
        for (int i = 0; i < stages && blockIdx.x + static_cast<long long>(i) * gridDim.x < turns; ++i)
            fill(blockIdx.x + static_cast<long long>(i) * gridDim.x, i);
    Vec8<T> w[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int c = (i * TPR + t) * 8;
        if (c < a.cols)
            w[i] = load8(static_cast<const T *>(a.weight) + c);
    }
    int n = 0, stage = 0;
    for (long long turn = blockIdx.x; turn < turns; turn += gridDim.x, ++n) {
        const bool ok = mbar_wait(&full[stage], (n / stages) & 1, a.err, kErrWaitV);
        const long long row = turn * ROWS + slot;
        float h[VPT][8];
        const uint8_t *from = ring + stage * stage_bytes + slot * pitch;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * TPR + t) * 8;
            if (c < a.cols) {
                unpack8(load8(reinterpret_cast<const T *>(from) + c), h[i]);
                if (res) {
                    float r[8];
                    unpack8(load8(reinterpret_cast<const T *>(from + ROWS * pitch) + c), r);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        h[i][e] += r[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    h[i][e] = 0.f;
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sum = fmaf(h[i][e], h[i][e], sum);
        sum = warp_sum(sum);
        if (threadIdx.x % 32 == 0)
            part[n & 1][threadIdx.x / 32] = sum;
        // Every thread has read the stage (and its row's parts are written).
        if (!__syncthreads_and(ok))
            break;
        const long long next = turn + static_cast<long long>(stages) * gridDim.x;
        if (threadIdx.x == 0 && next < turns)
            fill(next, stage);
        stage = stage + 1 == stages ? 0 : stage + 1;
        if (row >= a.rows) // whole warps: the last turn's missing rows
            continue;
        if (res) {
            T *to = static_cast<T *>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * TPR + t) * 8;
                if (c < a.cols)
                    store8(to + c, pack8<T>(h[i]));
            }
        }
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k)
            sum += part[n & 1][slot * WARPS + k];
        const float rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float wf[8];
            unpack8(w[i], wf);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                h[i][e] = (i * TPR + t) * 8 < a.cols ? h[i][e] * rstd * wf[e] : 0.f;
        }
        write_row<T, QUANT, TPR, VPT>(a, row, groups, t, h);
    }
    // After a wait that gave up: every copy lands before the CTA's memory goes.
    if (threadIdx.x == 0) {
        for (; n < filled; ++n) {
            const uint64_t start = globaltimer_ns();
            while (!mbar_try_wait(smem_u32(&full[n % stages]), (n / stages) & 1))
                if (globaltimer_ns() - start > kWaitLimitNs) {
                    atomicOr(a.err, kErrWaitDrain);
                    break;
                }
        }
    }
}

// Any alignment, up to 8192 columns: WARPS warps own a row, warp w its groups w, w +
// WARPS.. of 128 columns (GROUPS of them, in registers), a lane every 32nd element, so that
// loads of single elements are still whole sectors.  Each element is written by the thread
// that read it.
template <typename T, bool QUANT, int WARPS, int GROUPS>
__global__ void __launch_bounds__(256) rows_odd_kernel(const RowsArgs a) {
    constexpr int ROWS = 8 / WARPS;
    static_assert(WARPS == 1 || WARPS == 8, "a barrier is the CTA's");
    __shared__ float part[2][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32 % WARPS;
    const int groups = (a.cols + kGroup - 1) / kGroup;
    const T *weight = static_cast<const T *>(a.weight);
    const bool res = a.residual != nullptr;
    int turn = 0;
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    for (long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / (32 * WARPS); row < a.rows; row += step) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        float h[GROUPS][4];
        auto column = [&](int i, int e) { return (i * WARPS + warp) * kGroup + e * 32 + lane; };
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[i][e] = column(i, e) < a.cols ? to_float(x[column(i, e)]) : 0.f;
        if (res) {
            const T *from = static_cast<const T *>(a.residual) + row * a.residual_stride;
            T *to = static_cast<T *>(a.residual_out) + row * a.residual_out_stride;
            float r[GROUPS][4];
#pragma unroll
            for (int i = 0; i < GROUPS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    r[i][e] = column(i, e) < a.cols ? to_float(from[column(i, e)]) : 0.f;
#pragma unroll
            for (int i = 0; i < GROUPS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[i][e] += r[i][e];
                    if (column(i, e) < a.cols)
                        to[column(i, e)] = from_float<T>(h[i][e]);
                }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sum = fmaf(h[i][e], h[i][e], sum);
        sum = warp_sum(sum);
        if constexpr (WARPS > 1) { // two buffers, as in rows_kernel
            if (lane == 0)
                part[turn][warp] = sum;
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k)
                sum += part[turn][k];
            turn ^= 1;
        }
        const float rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[i][e] = column(i, e) < a.cols ? h[i][e] * rstd * to_float(weight[column(i, e)]) : 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int group = i * WARPS + warp;
            if (group >= groups)
                break;
            if constexpr (QUANT) {
                float amax = fmaxf(fmax3(fabsf(h[i][0]), fabsf(h[i][1]), fabsf(h[i][2])), fabsf(h[i][3]));
                amax = half_warp_max(amax);
                const float scale = group_scale(fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16)));
                const Divisor d = divisor_of(scale);
                if (lane == 0)
                    a.scales[row * groups + group] = scale;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (column(i, e) < a.cols)
                        static_cast<uint8_t *>(a.out)[row * a.out_stride + column(i, e)] =
                            static_cast<uint8_t>(e4m3x2(d.template quotient<false>(h[i][e]), 0.f));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (column(i, e) < a.cols)
                        static_cast<T *>(a.out)[row * a.out_stride + column(i, e)] = from_float<T>(h[i][e]);
            }
        }
    }
}

// One CTA per row; a warp takes a group of 128 columns, four elements a lane.
// Each element is written by the thread that read it last, so that an output
// may be the same tensor as x or the residual.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(256) rows_scalar_kernel(const RowsArgs a) {
    __shared__ float part[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int groups = (a.cols + kGroup - 1) / kGroup;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
        float rstd = 1.f;
        float sum = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += 256) {
            const float h = to_float(x[c]) + (res ? to_float(res[c]) : 0.f);
            sum = fmaf(h, h, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0)
            part[warp] = sum;
        __syncthreads();
        sum = 0.f;
        for (int k = 0; k < 8; ++k)
            sum += part[k];
        __syncthreads(); // before the next row's parts, and before a row that is written in place
        rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
        for (int g = warp; g < groups; g += 8) {
            float y[4], amax = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = g * kGroup + e * 32 + lane;
                y[e] = 0.f;
                if (c < a.cols) {
                    y[e] = to_float(x[c]);
                    if (res) {
                        y[e] += to_float(res[c]);
                        static_cast<T *>(a.residual_out)[row * a.residual_out_stride + c] = from_float<T>(y[e]);
                    }
                    y[e] = y[e] * rstd * to_float(static_cast<const T *>(a.weight)[c]);
                }
                amax = fmaxf(amax, fabsf(y[e]));
            }
            float scale = 1.f;
            if constexpr (QUANT) {
                amax = half_warp_max(amax);
                scale = group_scale(fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16)));
                if (lane == 0)
                    a.scales[row * groups + g] = scale;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = g * kGroup + e * 32 + lane;
                if (c >= a.cols)
                    continue;
                if constexpr (QUANT)
                    static_cast<uint8_t *>(a.out)[row * a.out_stride + c] =
                        static_cast<uint8_t>(e4m3x2(divisor_of(scale).template quotient<false>(y[e]), 0.f));
                else
                    static_cast<T *>(a.out)[row * a.out_stride + c] = from_float<T>(y[e]);
            }
        }
    }
}

// Eight elements from column c on by single loads, zeros past the row's end.
template <typename T> __device__ __forceinline__ void load8_any(const T *x, int c, int cols, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        f[e] = c + e < cols ? to_float(x[e]) : 0.f;
}
// Eight e4m3 values to column c on: at once where they are aligned and all in the row.
__device__ __forceinline__ void store8_e4m3(uint8_t *q, int c, int cols, bool aligned, uint2 v) {
    if (aligned && c + 8 <= cols) {
        *reinterpret_cast<uint2 *>(q) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols)
                q[e] = static_cast<uint8_t>((e < 4 ? v.x : v.y) >> (8 * (e % 4)) & 0xffu);
    }
}

// The largest of four magnitudes over the 16 lanes of a half warp: while lanes halve, so
// do the values that each still holds, and lane l ends with value l / 4 (5 shuffles, not
// 16; 24000 x 4096 56 -> 50 us, with one lane's division for each).
__device__ __forceinline__ float max_of_four(const float (&m)[4], int lane) {
    const bool high = lane & 8, odd = lane & 4;
    const float a = fmaxf(high ? m[2] : m[0], __shfl_xor_sync(0xffffffffu, high ? m[0] : m[2], 8));
    const float b = fmaxf(high ? m[3] : m[1], __shfl_xor_sync(0xffffffffu, high ? m[1] : m[3], 8));
    float v = fmaxf(odd ? b : a, __shfl_xor_sync(0xffffffffu, odd ? a : b, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
}

// Groups of 128 columns need nothing from the rest of their row, so that all groups of
// all rows are one list: a half warp takes a group, a warp runs of 8, in four steps.
// 24000 x 4096 bf16 49 us, 24000 x 1152 16 us; a row per CTA took 50 and 27 us:
// its threads past the row's end are idle.
constexpr int kSteps = 4;
// kWhole: rows of whole groups, one behind the other in x and in out.  kAny: rows that
// 16-byte loads cannot read, by single elements (24000 x 997 25 us, x 4097 86).
enum : int { kWhole, kPitched, kAny };
template <typename T, int MODE> __global__ void __launch_bounds__(256, 4) quantize_rows_kernel(const RowsArgs a, bool aligned) {
    constexpr bool WHOLE = MODE == kWhole;
    const int lane = threadIdx.x & 31, part = lane & 15, groups = (a.cols + kGroup - 1) / kGroup;
    const long long total = a.rows * groups;
    const long long begin = (blockIdx.x * 8ll + threadIdx.x / 32) * (2 * kSteps), stride = gridDim.x * 8ll * (2 * kSteps);
    // This half warp's group `at`, its row and its place in the row.
    long long at = begin + lane / 16, row = 0, rows_on = 0;
    int g = 0, groups_on = 0;
    if constexpr (!WHOLE) {
        row = at / groups;
        g = static_cast<int>(at - row * groups);
        rows_on = stride / groups;
        groups_on = static_cast<int>(stride - rows_on * groups);
    }
    const long long x_wrap = a.x_stride - static_cast<long long>(groups) * kGroup;
    const long long q_wrap = a.out_stride - static_cast<long long>(groups) * kGroup;
    for (long long first = begin; first < total; first += stride, at += stride) { // the whole warp
        float h[kSteps][8], top[kSteps];
        {
            Vec8<T> v[MODE == kAny ? 1 : kSteps];
            const T *x = static_cast<const T *>(a.x) + (WHOLE ? at * kGroup : row * a.x_stride + g * kGroup) + part * 8;
            int in = g;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int c = in * kGroup + part * 8;
                if constexpr (MODE == kAny) {
                    load8_any(x, c, at + 2 * i < total ? a.cols : 0, h[i]);
                } else {
                    v[i] = Vec8<T>{};
                    if (at + 2 * i < total && (WHOLE || c < a.cols))
                        v[i] = load8(x);
                }
                x += 2 * kGroup;
                if constexpr (!WHOLE)
                    for (in += 2; in >= groups; in -= groups)
                        x += x_wrap;
            }
            if constexpr (MODE != kAny) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
                    unpack8(v[i], h[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            top[i] = amax8(h[i]);
        // A lane divides for one step and hands the result round.
        constexpr int LANES = 16 / kSteps;
        const float scale = group_scale(max_of_four(top, part));
        const Divisor divisor = divisor_of(scale);
        const long long own = at + 2 * (part / LANES);
        if (part % LANES == 0 && own < total)
            a.scales[own] = scale;
        uint8_t *q = static_cast<uint8_t *>(a.out) + (WHOLE ? at * kGroup : row * a.out_stride + g * kGroup) + part * 8;
        int in = g;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            Divisor d;
            d.scale = __shfl_sync(0xffffffffu, divisor.scale, i * LANES, 16);
            d.inv = __shfl_sync(0xffffffffu, divisor.inv, i * LANES, 16);
            const int c = in * kGroup + part * 8;
            if constexpr (MODE == kAny)
                store8_e4m3(q, c, at + 2 * i < total ? a.cols : 0, aligned, e4m3x8<true>(h[i], d));
            else if (at + 2 * i < total && (WHOLE || c < a.cols))
                *reinterpret_cast<uint2 *>(q) = e4m3x8<true>(h[i], d);
            q += 2 * kGroup;
            if constexpr (!WHOLE)
                for (in += 2; in >= groups; in -= groups)
                    q += q_wrap;
        }
        if constexpr (!WHOLE) {
            row += rows_on;
            g += groups_on;
            if (g >= groups) {
                g -= groups;
                ++row;
            }
        }
    }
}

// One CTA per 128 x 128 block: thread = 8 columns of every 16th row, its 64
// elements in registers between the largest magnitude and the conversion.
// 24000 x 4096 bf16 52 us; without VEC (by single elements) 24000 x 4095 144 us.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T *x, uint8_t *q, float *scales, long long rows,
                                                              int cols, long long x_stride, long long q_stride,
                                                              bool aligned) {
    __shared__ float part[8];
    const int c = blockIdx.x * kGroup + (threadIdx.x % 16) * 8;
    const long long r0 = static_cast<long long>(blockIdx.y) * kGroup + threadIdx.x / 16;
    float f[8][8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + i * 16;
        if constexpr (VEC) {
            Vec8<T> v{};
            if (r < rows && c < cols)
                v = load8(x + r * x_stride + c);
            unpack8(v, f[i]);
        } else {
            load8_any(x + r * x_stride + c, c, r < rows ? cols : 0, f[i]);
        }
        amax = fmaxf(amax, amax8(f[i]));
    }
    amax = half_warp_max(amax);
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
    if (threadIdx.x % 32 == 0)
        part[threadIdx.x / 32] = amax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k)
        amax = fmaxf(amax, part[k]);
    const float scale = group_scale(amax);
    const Divisor divisor = divisor_of(scale);
    if (threadIdx.x == 0)
        scales[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + i * 16;
        if (r < rows)
            store8_e4m3(q + r * q_stride + c, c, cols, aligned, e4m3x8<true>(f[i], divisor));
    }
}

template <typename T, bool QUANT, int TPR, int VPT, int ROWS>
int launch_rows(const RowsArgs &a, cudaStream_t stream) {
    // As many CTAs as run at once: every one takes the same number of rows, +-1.
    static std::atomic<int> resident{0};
    int each = resident.load(std::memory_order_relaxed);
    if (!each) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, rows_kernel<T, QUANT, TPR, VPT, ROWS>,
                                                          TPR * ROWS, 0) != cudaSuccess ||
            each < 1)
            each = 1;
        resident.store(each, std::memory_order_relaxed);
    }
    const long long ctas = (a.rows + ROWS - 1) / ROWS;
    const long long most = static_cast<long long>(fmha_sm_count()) * each;
    rows_kernel<T, QUANT, TPR, VPT, ROWS>
        <<<static_cast<unsigned>(std::min(ctas, most)), TPR * ROWS, 0, stream>>>(a);
    return static_cast<int>(cudaGetLastError());
}

template <typename T, bool QUANT, int TPR, int VPT> int launch_stream(const RowsArgs &a, cudaStream_t stream) {
    constexpr int ROWS = kStreamThreads / TPR;
    const int stage = ROWS * a.cols * static_cast<int>(sizeof(T)) * (a.residual ? 2 : 1);
    const int stages = std::max(2, std::min(kMaxStages, kStreamBytes / stage));
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(rows_stream_kernel<T, QUANT, TPR, VPT>),
                                         std::max(kStreamBytes, 2 * 1024 * 8 * static_cast<int>(sizeof(T)) * 2), done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    const long long turns = (a.rows + ROWS - 1) / ROWS;
    const int each = 200 * 1024 / (stages * stage); // CTAs on an SM
    const long long most = static_cast<long long>(fmha_sm_count()) * std::max(1, std::min(each, 4));
    rows_stream_kernel<T, QUANT, TPR, VPT>
        <<<static_cast<unsigned>(std::min(turns, most)), kStreamThreads, stages * stage, stream>>>(a, stages);
    return static_cast<int>(cudaGetLastError());
}

template <typename T, bool QUANT, int WARPS, int GROUPS>
int launch_odd(const RowsArgs &a, cudaStream_t stream) {
    constexpr int ROWS = 8 / WARPS;
    const long long ctas = std::min((a.rows + ROWS - 1) / ROWS, 8ll * fmha_sm_count());
    rows_odd_kernel<T, QUANT, WARPS, GROUPS><<<static_cast<unsigned>(ctas), 256, 0, stream>>>(a);
    return static_cast<int>(cudaGetLastError());
}

// Rows of `vecs` 8-element vectors.
template <typename T, bool QUANT> int launch_norm(const RowsArgs &a, int vecs, cudaStream_t stream) {
    // Wide rows, and enough of them for every SM to keep its ring busy.  Measured (bf16,
    // residual, e4m3): 16384 x 8192 148 us against rows_kernel's 176, 16384 x 4096 83 and
    // 104, 23328 x 2048 65 and 79 (a warp for each row).  Narrower rows leave a ring less
    // than a warp for each row gains: 23328 x 1024 38 and 30, 23328 x 512 26 and 20.
    if (vecs > 192 && vecs <= 1024 && a.rows * vecs >= 64ll * 1024 * 8) {
        if (vecs <= 256)
            return launch_stream<T, QUANT, 64, 4>(a, stream);
        if (vecs <= 512)
            return launch_stream<T, QUANT, 128, 4>(a, stream);
        return launch_stream<T, QUANT, 256, 4>(a, stream);
    }
    if (vecs <= 32)
        return launch_rows<T, QUANT, 32, 1, 4>(a, stream);
    if (vecs <= 64)
        return launch_rows<T, QUANT, 32, 2, 4>(a, stream);
    if (vecs <= 128)
        return launch_rows<T, QUANT, 32, 4, 4>(a, stream);
    if (vecs <= 160) // 23328 x 1152 38 us; without the next row's loads 47, by 128 threads to a row 57
        return launch_rows<T, QUANT, 32, 5, 4>(a, stream);
    if (vecs <= 192)
        return launch_rows<T, QUANT, 32, 6, 4>(a, stream);
    if (vecs <= 256)
        return launch_rows<T, QUANT, 128, 2, 1>(a, stream);
    if (vecs <= 512)
        return launch_rows<T, QUANT, 128, 4, 1>(a, stream);
    if (vecs <= 1024)
        return launch_rows<T, QUANT, 256, 4, 1>(a, stream);
    return launch_rows<T, QUANT, 512, 4, 1>(a, stream);
}

template <typename T> int launch_quantize(const RowsArgs &a, cudaStream_t stream) {
    constexpr int kAlign = 16 / sizeof(T); // elements of 16 bytes
    const bool aligned = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && a.out_stride % 8 == 0;
    const bool vec = aligned && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.cols % 8 == 0 && a.x_stride % kAlign == 0;
    const long long runs = (a.rows * ((a.cols + kGroup - 1) / kGroup) + 2 * kSteps - 1) / (2 * kSteps);
    const unsigned grid = static_cast<unsigned>(std::min((runs + 7) / 8, 4ll * fmha_sm_count()));
    // Without rows to keep track of: 24000 x 4096 49 us, with them 52.
    if (vec && a.cols % kGroup == 0 && a.x_stride == a.cols && a.out_stride == a.cols)
        quantize_rows_kernel<T, kWhole><<<grid, 256, 0, stream>>>(a, aligned);
    else if (vec)
        quantize_rows_kernel<T, kPitched><<<grid, 256, 0, stream>>>(a, aligned);
    else
        quantize_rows_kernel<T, kAny><<<grid, 256, 0, stream>>>(a, aligned);
    return static_cast<int>(cudaGetLastError());
}

template <typename T, bool QUANT> int launch_typed(const RowsArgs &a, cudaStream_t stream) {
    constexpr int kAlign = 16 / sizeof(T);
    const uintptr_t base = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                           reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.residual_out);
    const uintptr_t out = reinterpret_cast<uintptr_t>(a.out);
    const bool vec = base % 16 == 0 && a.cols % 8 == 0 && a.x_stride % kAlign == 0 &&
                     (!a.residual || (a.residual_stride % kAlign == 0 && a.residual_out_stride % kAlign == 0)) &&
                     (QUANT ? out % 8 == 0 && a.out_stride % 8 == 0 : out % 16 == 0 && a.out_stride % kAlign == 0);
    const int vecs = a.cols / 8;
    if (vec && vecs <= 2048)
        return launch_norm<T, QUANT>(a, vecs, stream);
    // 17679 x 3727 bf16, residual, e4m3 129 us, 251 by rows_scalar_kernel; 60000 x 412 57
    // and 158; 16000 x 8001 299 and 458.
    if (a.cols <= 512)
        return launch_odd<T, QUANT, 1, 4>(a, stream);
    if (a.cols <= 1024)
        return launch_odd<T, QUANT, 1, 8>(a, stream);
    if (a.cols <= 2048)
        return launch_odd<T, QUANT, 8, 2>(a, stream);
    if (a.cols <= 4096)
        return launch_odd<T, QUANT, 8, 4>(a, stream);
    if (a.cols <= 8192)
        return launch_odd<T, QUANT, 8, 8>(a, stream);
    const unsigned grid = static_cast<unsigned>(std::min<long long>(a.rows, 8ll * fmha_sm_count()));
    rows_scalar_kernel<T, QUANT><<<grid, 256, 0, stream>>>(a);
    return static_cast<int>(cudaGetLastError());
}

template <typename T> int launch_dtype(const RowsArgs &a, cudaStream_t stream) {
    if (!a.norm)
        return launch_quantize<T>(a, stream);
    return a.quantize ? launch_typed<T, true>(a, stream) : launch_typed<T, false>(a, stream);
}

template <typename T>
int launch_blocks(const T *x, uint8_t *q, float *scales, long long rows, int cols, long long x_stride,
                  long long q_stride, cudaStream_t stream) {
    const dim3 grid((cols + kGroup - 1) / kGroup, static_cast<unsigned>((rows + kGroup - 1) / kGroup));
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && cols % 8 == 0 &&
                     x_stride % (16 / static_cast<int>(sizeof(T))) == 0;
    const bool aligned = reinterpret_cast<uintptr_t>(q) % 8 == 0 && q_stride % 8 == 0;
    if (vec)
        quantize_blocks_kernel<T, true><<<grid, 256, 0, stream>>>(x, q, scales, rows, cols, x_stride, q_stride, aligned);
    else
        quantize_blocks_kernel<T, false><<<grid, 256, 0, stream>>>(x, q, scales, rows, cols, x_stride, q_stride, aligned);
    return static_cast<int>(cudaGetLastError());
}

} // namespace

int rows_launch(const RowsArgs &a, cudaStream_t stream) {
    switch (a.dtype) {
    case kF32:
        return launch_dtype<float>(a, stream);
    case kBF16:
        return launch_dtype<__nv_bfloat16>(a, stream);
    default:
        return launch_dtype<__half>(a, stream);
    }
}

int quantize_blocks_launch(const void *x, void *q, float *scales, long long rows, int cols, long long x_stride,
                           long long q_stride, int dtype, cudaStream_t stream) {
    uint8_t *to = static_cast<uint8_t *>(q);
    switch (dtype) {
    case kF32:
        return launch_blocks(static_cast<const float *>(x), to, scales, rows, cols, x_stride, q_stride, stream);
    case kBF16:
        return launch_blocks(static_cast<const __nv_bfloat16 *>(x), to, scales, rows, cols, x_stride, q_stride, stream);
    default:
        return launch_blocks(static_cast<const __half *>(x), to, scales, rows, cols, x_stride, q_stride, stream);
    }
}

} // namespace omni_b200
