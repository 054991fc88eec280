// rotary.cu -- rotary positions with one or more axes, for q and k in one launch.
//
// Pair i of a head's columns, (x0, x1) = (x[i], x[i + pairs]) or (x[2i], x[2i + 1]), is
// turned by angle = positions[axes[i], b, t] * frequencies[i]:
//   y0 = x0 cos - x1 sin,  y1 = x1 cos + x0 sin   (inverse, the backward pass: -sin).
// The angle of a far position needs more than fp32: its product, its share of a whole
// turn and the subtraction of the whole turns are fp64, the fraction that is left
// becomes fp32 for sincospif (its error is below 2^-24 of a turn).
//
// The bound is the memory traffic: each element is read and written once.  A thread
// holds the sines and cosines of V pairs of one token in registers and goes over heads, so
// that they are computed once for all heads of its group (gridDim.y groups); neighbouring
// threads take neighbouring columns, then tokens, so rows are read whole whatever the layout.
// 8192 tokens x 40 heads of 128 in bf16: 35.1 us, 4.8 TB/s with the launch; without angles it
// would take 31.  fp32 angles would save nothing.  In fp32: 58 us, 5.8 TB/s.
#include "e4m3.cuh"
#include "layer.h"

#include <algorithm>

namespace omni_b200 {
namespace {

constexpr int kThreads = 256, kRuns = 4;
// Threads of an SM that heads are split for.  More than fit: the kernel of eight pairs has 54
// registers, 1024 threads an SM, so that 8192 tokens x 40 heads of 128 make 1280 CTAs in 592
// places, 2.2 rounds, and compute each angle five times.
constexpr long long kFull = 2048;

struct RotaryParams {
    const void *x[2]; // q, k
    void *y[2];
    long long xs[2][3], ys[2][3]; // batch, head, token
    const void *positions, *frequencies;
    long long ps[3]; // axis, batch, token
    long long items, tail_items;
    unsigned pair_blocks;
    int heads, all_heads; // of q; of q and k
    int tokens, hd, pairs, chunks, tail; // chunks: of V pairs; tail: of V columns that are copied
    int position_type;
    bool frequency_f64;
    float sign;
    uint8_t axes[kMaxPairs];
};

template <typename T, int N> struct alignas(sizeof(T) * N) Run {
    T e[N];
};

__device__ __forceinline__ double position_at(const RotaryParams &p, long long at) {
    if (p.position_type == kPositionI32)
        return static_cast<const int *>(p.positions)[at];
    if (p.position_type == kPositionI64)
        return static_cast<double>(static_cast<const long long *>(p.positions)[at]);
    return static_cast<const float *>(p.positions)[at];
}

// Elements of a load where a thread has v pairs: what every row has to be aligned to.
__host__ __device__ constexpr int run_length(int v, bool adjacent, int size) {
    const int n = adjacent ? 2 * v : v;
    return v == 1 ? 1 : n * size > 16 ? 16 / size : n;
}

// V pairs a thread.
template <typename T, int V, bool ADJACENT> __global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    // The pairs' CTAs, then those of the columns behind them (in one warp they would wait for
    // each other: 8192 tokens x 40 heads of 128 with 16 pairs 55 us, 36 so).
    const bool behind = blockIdx.x >= p.pair_blocks;
    const long long item = static_cast<long long>(blockIdx.x - (behind ? p.pair_blocks : 0)) * kThreads + threadIdx.x;
    if (item >= (behind ? p.tail_items : p.items))
        return;
    const int per_token = behind ? p.tail : p.chunks;
    const long long token = item / per_token; // of all sequences
    const int chunk = static_cast<int>(item - token * per_token);
    const long long b = token / p.tokens, t = token - b * p.tokens;
    if (behind) {
        const int col = 2 * p.pairs + chunk * V;
        using R = Run<T, V>;
        for (int h0 = blockIdx.y * kRuns; h0 < p.all_heads; h0 += gridDim.y * kRuns) {
            R r[kRuns];
#pragma unroll
            for (int u = 0; u < kRuns; ++u) {
                const int h = min(h0 + u, p.all_heads - 1), w = h >= p.heads, hh = h - (w ? p.heads : 0);
                r[u] = *reinterpret_cast<const R *>(static_cast<const T *>(p.x[w]) + b * p.xs[w][0] + hh * p.xs[w][1] + t * p.xs[w][2] + col);
            }
#pragma unroll
            for (int u = 0; u < kRuns; ++u) {
                const int h = h0 + u, w = h >= p.heads, hh = h - (w ? p.heads : 0);
                if (h < p.all_heads)
                    *reinterpret_cast<R *>(static_cast<T *>(p.y[w]) + b * p.ys[w][0] + hh * p.ys[w][1] + t * p.ys[w][2] + col) = r[u];
            }
        }
        return;
    }
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int pair = chunk * V + i;
        const double f = p.frequency_f64 ? static_cast<const double *>(p.frequencies)[pair]
                                         : static_cast<const float *>(p.frequencies)[pair];
        const double turns = position_at(p, p.axes[pair] * p.ps[0] + b * p.ps[1] + t * p.ps[2]) * f * 0.15915494309189535;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn[i], &cs[i]);
        sn[i] *= p.sign;
    }
    // Runs of at most 16 bytes: halves are V elements each, adjacent pairs 2 V together.  A
    // single pair (V = 1) goes element by element: rows may lie at any address of the type.
    constexpr int N = ADJACENT ? 2 * V : V, L = run_length(V, ADJACENT, sizeof(T));
    using R = Run<T, L>;
    constexpr int P = N / L; // runs of one piece
    constexpr int PIECES = ADJACENT ? 1 : 2;
    const int col = chunk * N;
    // Four runs, of up to four heads, are read before any is written (the outputs may be
    // the inputs, so the compiler would not move a read over a write): 8192 tokens x 40 heads of
    // 128 34 us, 36 with two runs; 32 x 729 tokens x 32 heads of 72 40 and 44.
    constexpr int HEADS = PIECES * P >= kRuns ? 1 : kRuns / (PIECES * P);
    for (int h0 = blockIdx.y * HEADS; h0 < p.all_heads; h0 += gridDim.y * HEADS) {
        R r[HEADS][PIECES * P];
#pragma unroll
        for (int u = 0; u < HEADS; ++u) {
            const int h = min(h0 + u, p.all_heads - 1), w = h >= p.heads, hh = h - (w ? p.heads : 0);
            const T *x = static_cast<const T *>(p.x[w]) + b * p.xs[w][0] + hh * p.xs[w][1] + t * p.xs[w][2] + col;
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int j = 0; j < P; ++j)
                    r[u][i * P + j] = *reinterpret_cast<const R *>(x + i * p.pairs + j * L);
        }
#pragma unroll
        for (int u = 0; u < HEADS; ++u) {
            const int h = h0 + u, w = h >= p.heads, hh = h - (w ? p.heads : 0);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int i0 = ADJACENT ? 2 * i : i, i1 = ADJACENT ? 2 * i + 1 : V + i;
                T &e0 = r[u][i0 / L].e[i0 % L], &e1 = r[u][i1 / L].e[i1 % L];
                const float x0 = to_float(e0), x1 = to_float(e1);
                e0 = from_float<T>(x0 * cs[i] - x1 * sn[i]);
                e1 = from_float<T>(x1 * cs[i] + x0 * sn[i]);
            }
            if (h < p.all_heads) {
                T *y = static_cast<T *>(p.y[w]) + b * p.ys[w][0] + hh * p.ys[w][1] + t * p.ys[w][2] + col;
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
#pragma unroll
                    for (int j = 0; j < P; ++j)
                        *reinterpret_cast<R *>(y + i * p.pairs + j * L) = r[u][i * P + j];
            }
        }
    }
}

template <typename T, int V> int launch_v(RotaryParams &p, long long rows, bool adjacent, bool in_place, cudaStream_t stream) {
    p.chunks = p.pairs / V;
    p.tail = in_place ? 0 : (p.hd - 2 * p.pairs) / V;
    p.items = rows * p.chunks;
    p.tail_items = rows * p.tail;
    const long long pair_blocks = (p.items + kThreads - 1) / kThreads;
    const long long blocks = pair_blocks + (p.tail_items + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffll)
        return static_cast<int>(cudaErrorInvalidValue);
    p.pair_blocks = static_cast<unsigned>(pair_blocks);
    // Heads are split over CTAs until every SM has its threads.
    const long long full = kFull / kThreads * fmha_sm_count();
    const int groups = static_cast<int>(std::min<long long>(p.all_heads, std::max<long long>(1, (full + blocks - 1) / blocks)));
    const dim3 grid(static_cast<unsigned>(blocks), groups);
    if (adjacent)
        rotary_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(p);
    else
        rotary_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

template <typename T> int launch_typed(RotaryParams &p, const RotaryArgs &a, bool in_place, cudaStream_t stream) {
    // The widest run that every row allows.
    auto fits = [&](int v) {
        const int n = run_length(v, a.adjacent, sizeof(T));
        if (a.pairs % v || (a.hd - 2 * a.pairs) % v)
            return false;
        for (int w = 0; w < (a.k ? 2 : 1); ++w) {
            const void *ends[2] = {w ? a.k : a.q, w ? a.k_out : a.q_out};
            const long long *strides[2] = {w ? a.ks : a.qs, w ? a.kos : a.qos};
            for (int i = 0; i < 2; ++i) {
                if (reinterpret_cast<uintptr_t>(ends[i]) % (n * sizeof(T)))
                    return false;
                for (int d = 0; d < 3; ++d)
                    if (strides[i][d] % n)
                        return false;
            }
        }
        return true;
    };
    const long long rows = static_cast<long long>(a.batch) * a.tokens;
    if (sizeof(T) == 2 && fits(8))
        return launch_v<T, sizeof(T) == 2 ? 8 : 4>(p, rows, a.adjacent, in_place, stream);
    if (fits(4))
        return launch_v<T, 4>(p, rows, a.adjacent, in_place, stream);
    return launch_v<T, 1>(p, rows, a.adjacent, in_place, stream);
}

} // namespace

int rotary_launch(const RotaryArgs &a, cudaStream_t stream) {
    RotaryParams p{};
    p.x[0] = a.q;
    p.x[1] = a.k;
    p.y[0] = a.q_out;
    p.y[1] = a.k_out;
    for (int d = 0; d < 3; ++d) {
        p.xs[0][d] = a.qs[d];
        p.xs[1][d] = a.ks[d];
        p.ys[0][d] = a.qos[d];
        p.ys[1][d] = a.kos[d];
        p.ps[d] = a.ps[d];
    }
    p.positions = a.positions;
    p.frequencies = a.frequencies;
    p.heads = a.heads;
    p.all_heads = a.heads + (a.k ? a.kv_heads : 0);
    p.tokens = a.tokens;
    p.hd = a.hd;
    p.pairs = a.pairs;
    p.position_type = a.position_type;
    p.frequency_f64 = a.frequency_f64;
    p.sign = a.inverse ? -1.f : 1.f;
    if (a.axes)
        std::copy(a.axes, a.axes + a.pairs, p.axes);
    const bool in_place = a.q == a.q_out && (!a.k || a.k == a.k_out);
    if (a.dtype == kF32)
        return launch_typed<float>(p, a, in_place, stream);
    if (a.dtype == kBF16)
        return launch_typed<__nv_bfloat16>(p, a, in_place, stream);
    return launch_typed<__half>(p, a, in_place, stream);
}

} // namespace omni_b200
