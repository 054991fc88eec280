// window_prompt_sm100.cu -- sliding-window attention for prompts and encoders on
// B200 (sm_100a).
//
// softmax(scale * q k^T + mask) v for blocks of 128 query rows.  A window leaves a
// block few keys, so a block is over after some ten steps, and its own chain
// (product, softmax, product) leaves the SM idle between them.  Each CTA therefore
// runs several blocks at once as independent chains, each with queries, keys,
// values, tensor memory and warps of its own: while one waits, another's
// exponentials use the MUFU (the bound: 16 per clock and SM).  Keys come 64 at a
// time, starting at the block's first visible key.
//   NC = 1 (head_dim <= 64): 3 chains, TMEM per chain S [0, 64), P [64, 96),
//     O [96, 160).
//   NC = 2 (head_dim <= 128): 2 chains, TMEM per chain S0, S1 [0, 128), O
//     [128, 256); P (16-bit pairs) over the first 32 columns of its S.
// Either way the next scores are computed while the softmax works on these: with
// one S as soon as the softmax has it in registers, with two at once.
//
// Per chain: 4 softmax warps (a row per thread = TMEM lane), one warp that finds the
// blocks and loads (TMA), and one that issues the tensor cores' products.  The
// loader publishes each block's description in shared memory, ahead of its use: the
// divisions and the reads of the lengths stay off the other warps' path.
// Exponentials are taken to base 2 with the scale folded in, statistics are fp32; a
// row keeps a stale maximum until it grows by more than 2^8, so that P <= 2^8 and O
// is rarely rescaled.  Two barriers tell that O has the product of step g (g & 1): a
// waiter may be a step behind the products, and one barrier's parity would mistake
// the step before the last for the one awaited.
//
// Tiles hold 64 columns (128 bytes, 128-byte swizzle) per row and chunk; columns
// past head_dim and rows past the tensor are TMA's zero fill.  Rows of v past a
// sequence's keys are cleared in shared memory (a NaN there would survive P = 0).
#include "fmha.h"
#include "sm100.cuh"
#include "tma.h"

#include <algorithm>
#include <cmath>

namespace omni_b200 {
namespace {

constexpr int kKeys = 64;    // keys of a step
constexpr int kMaxBatch = 496; // sequences that the item table holds

struct PromptParams {
    CUtensorMap tq, tk, tv;
    void *out;
    long long o_sb, o_sh, o_st;
    const int *lengths, *q_lengths;
    int batch, heads, group, q_len, kv_len, hd;
    int window, right, sinks;
    int out_dtype, out_vec, table;
    float scale_log2;
    int *err;
};

template <int NC> struct PromptShape {
    static constexpr int CHAINS = NC == 1 ? 3 : 2;
    static constexpr int STAGES = NC == 1 ? 3 : 2; // of keys, and of values
    static constexpr int SOFT_WARPS = CHAINS * 4, ISSUE_WARP = SOFT_WARPS + CHAINS;
    static constexpr int THREADS = (SOFT_WARPS + 2 * CHAINS + 3) / 4 * 128; // whole warpgroups
    // Registers: 640 x 96 at launch = 384 x 112 + 256 x 72; 384 x 168 = 256 x 216 + 128 x 72.
    static constexpr int SOFT_REGS = NC == 1 ? 112 : 216, CONTROL_REGS = 72;
    static constexpr int Q_BYTES = NC * 128 * 128, KV_BYTES = NC * kKeys * 128;
    static constexpr int CHAIN_BYTES = Q_BYTES + 2 * STAGES * KV_BYTES;
    static constexpr uint32_t COLS = NC == 1 ? 160 : 256, O_COL = NC == 1 ? 96 : 128;
    static constexpr int BARS = 26, BLOCK_INTS = 12; // per chain; per published block (two of them)
    static constexpr int TABLE_BYTES = (2 * kMaxBatch + 1) * 4;
    static constexpr int SMEM = CHAINS * (CHAIN_BYTES + BARS * 8 + 2 * BLOCK_INTS * 4) + 16 + TABLE_BYTES + 1024;
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};

template <int N> __device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int *err, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}
// Bounded by time only: nothing may be in flight when the CTA ends.
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
// One arrive per warp, after its lanes.
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
        mbar_arrive(bar);
}
template <bool BF16> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// 128 query rows of one (sequence, head): steps of 64 keys, first those that hold
// sinks before the window ([0, sink_steps)), then from key `base` on.
struct Block {
    int b, h, q0, n, rows, pos0;
    int sink_steps, base, steps;
    bool skip; // no rows
};

__device__ __forceinline__ int held_keys(const PromptParams &p, int b) {
    return p.lengths ? max(0, min(p.lengths[b], p.kv_len)) : p.kv_len;
}
__device__ __forceinline__ int held_rows(const PromptParams &p, int b) {
    return p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
}

// Block u of a chain: round k = u / chains goes through the chains forwards and
// backwards in turn.  Blocks of ragged batches come from the table (sequences with
// most keys first, `pre` blocks before each), others with the last rows first, so
// that without a window the longest start first.
__device__ __forceinline__ Block block_at(const PromptParams &p, const int *table, int u, int chains) {
    const int k = u / chains, c = u - k * chains, r = k * chains + ((k & 1) ? chains - 1 - c : c);
    Block it;
    if (p.table) {
        const int *seq = table, *pre = table + kMaxBatch;
        if (r >= pre[p.batch]) {
            it.b = it.h = it.q0 = it.n = it.rows = it.pos0 = it.sink_steps = it.base = it.steps = 0;
            it.skip = true;
            return it;
        }
        int from = 0, to = p.batch - 1; // last rank with pre[rank] <= r
        while (from < to) {
            const int mid = (from + to + 1) >> 1;
            if (pre[mid] <= r)
                from = mid;
            else
                to = mid - 1;
        }
        const int off = r - pre[from], blocks = (pre[from + 1] - pre[from]) / p.heads;
        it.b = seq[from];
        it.h = off % p.heads;
        it.q0 = (blocks - 1 - off / p.heads) * 128;
    } else {
        const int per = p.batch * p.heads, block = r / per, bh = r - block * per;
        it.q0 = ((p.q_len + 127) / 128 - 1 - block) * 128;
        it.b = bh / p.heads;
        it.h = bh - it.b * p.heads;
    }
    it.n = held_keys(p, it.b);
    it.rows = held_rows(p, it.b);
    it.pos0 = it.n - it.rows;
    it.skip = it.q0 < 0 || it.q0 >= it.rows;
    const int first = it.pos0 + it.q0, last = it.pos0 + min(it.q0 + 127, it.rows - 1);
    const int high = it.skip ? 0 : max(0, min(it.n, last + p.right + 1));
    const int low = p.window > 0 ? max(0, min(first - p.window + 1, high)) : 0;
    it.sink_steps = (min(p.sinks, low) + kKeys - 1) / kKeys;
    it.base = max(low, it.sink_steps * kKeys);
    it.steps = it.sink_steps + max(0, high - it.base + kKeys - 1) / kKeys;
    return it;
}

// First key of step j.
__device__ __forceinline__ int step_key(int j, int sink_steps, int base) {
    return j * kKeys + (j < sink_steps ? 0 : base - sink_steps * kKeys);
}

template <int NC, bool BF16>
__global__ void __launch_bounds__(PromptShape<NC>::THREADS, 1) window_prompt_kernel(const __grid_constant__ PromptParams p) {
    using S = PromptShape<NC>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *all_bars = reinterpret_cast<uint64_t *>(smem + S::CHAINS * S::CHAIN_BYTES);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(all_bars + S::CHAINS * S::BARS);
    int *published = reinterpret_cast<int *>(tmem_holder + 4); // [chain][2][BLOCK_INTS]
    int *table = published + S::CHAINS * 2 * S::BLOCK_INTS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err = p.err;

    if (p.table) {
        int *seq = table, *pre = table + kMaxBatch;
        for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
            const int mine = held_keys(p, b);
            int rank = 0;
            for (int o = 0; o < p.batch; ++o) {
                const int its = held_keys(p, o);
                rank += its > mine || (its == mine && o < b) ? 1 : 0;
            }
            seq[rank] = b;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int sum = 0;
            for (int r = 0; r < p.batch; ++r) {
                pre[r] = sum;
                sum += p.heads * ((held_rows(p, seq[r]) + 127) / 128);
            }
            pre[p.batch] = sum;
        }
    }
    if (threadIdx.x == 0) {
        for (int c = 0; c < S::CHAINS; ++c) {
            uint64_t *bar = all_bars + c * S::BARS;
            for (int i = 0; i < S::BARS; ++i)
                mbar_init(&bar[i], i >= 24 ? 5 : i >= 19 && i < 22 ? 4 : 1);
        }
        fence_mbarrier_init();
    }
    if (warp == S::ISSUE_WARP) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    const int chain = warp < S::SOFT_WARPS ? warp / 4 : (warp - S::SOFT_WARPS) % S::CHAINS;
    // Chain c of every CTA before chain c + 1 of any: few blocks spread over the SMs.
    const int chains = gridDim.x * S::CHAINS, mine = chain * gridDim.x + blockIdx.x;
    const int per_block = p.table ? table[kMaxBatch + p.batch] : p.batch * p.heads * ((p.q_len + 127) / 128);
    const int blocks = (per_block + chains - 1) / chains * chains; // whole rounds: their last may be empty
    uint8_t *sq = smem + chain * S::CHAIN_BYTES, *sk = sq + S::Q_BYTES, *sv = sk + S::STAGES * S::KV_BYTES;
    uint64_t *bar = all_bars + chain * S::BARS;
    uint64_t *q_full = bar, *q_empty = bar + 1, *k_full = bar + 2, *k_empty = bar + 5, *v_full = bar + 8,
             *v_empty = bar + 11, *s_full = bar + 14, *pv_done = bar + 16, *drain = bar + 18;
    uint64_t *p_full = bar + 19, *o_free = bar + 20, *s_free = bar + 21; // an arrive of each softmax warp
    uint64_t *block_full = bar + 22, *block_empty = bar + 24;            // [2]; read by five warps
    static_assert(S::STAGES <= 3, "barrier places");
    int *mine_published = published + chain * 2 * S::BLOCK_INTS;
    const uint32_t tm = tmem + chain * S::COLS;

    if (warp >= S::SOFT_WARPS) {
        reg_dec<S::CONTROL_REGS>();
        if (warp < S::ISSUE_WARP) {
            // ------------------------------------------------- blocks and loads
            int nk = 0, nv = 0, items = 0, listed = 0;
            bool ok = true;
            auto publish = [&](const Block &it) {
                const int slot = listed & 1;
                if (!warp_wait(&block_empty[slot], ((listed >> 1) & 1) ^ 1, err, kErrWaitEmpty))
                    return false;
                if (lane == 0) {
                    int *to = mine_published + slot * S::BLOCK_INTS;
                    to[0] = it.b, to[1] = it.h, to[2] = it.q0, to[3] = it.n, to[4] = it.rows;
                    to[5] = it.sink_steps, to[6] = it.base, to[7] = it.steps;
                    mbar_arrive(&block_full[slot]);
                }
                __syncwarp();
                ++listed;
                return true;
            };
            auto load = [&](uint8_t *to, const CUtensorMap *map, uint64_t *full, uint64_t *empty, int &n, int key, int head, int b) {
                const int st = n % S::STAGES;
                if (!warp_wait(&empty[st], ((n / S::STAGES) & 1) ^ 1, err, kErrWaitEmpty))
                    return false;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[st], S::KV_BYTES);
                    for (int c = 0; c < NC; ++c)
                        tma_load_4d(to + st * S::KV_BYTES + c * kKeys * 128, map, &full[st], c * 64, key, head, b);
                }
                __syncwarp();
                ++n;
                return true;
            };
            for (int u = mine; ok && u < blocks; u += chains) {
                const Block it = block_at(p, table, u, chains);
                if (it.skip)
                    continue;
                if (!(ok = publish(it)))
                    break;
                if (it.steps == 0)
                    continue;
                const int head = it.h / p.group;
                if (!(ok = warp_wait(q_empty, (items & 1) ^ 1, err, kErrWaitEmpty)))
                    break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(q_full, S::Q_BYTES);
                    for (int c = 0; c < NC; ++c)
                        tma_load_4d(sq + c * 128 * 128, &p.tq, q_full, c * 64, it.q0, it.h, it.b);
                }
                __syncwarp();
                ++items;
                // Keys a step ahead of values: they are wanted a step earlier.
                ok = load(sk, &p.tk, k_full, k_empty, nk, step_key(0, it.sink_steps, it.base), head, it.b);
                for (int j = 0; ok && j < it.steps; ++j) {
                    if (j + 1 < it.steps)
                        ok = load(sk, &p.tk, k_full, k_empty, nk, step_key(j + 1, it.sink_steps, it.base), head, it.b);
                    ok = ok && load(sv, &p.tv, v_full, v_empty, nv, step_key(j, it.sink_steps, it.base), head, it.b);
                }
            }
            if (ok) {
                Block end{};
                end.steps = -1;
                publish(end);
            }
            // Every copy lands before the CTA ends.
            if (items > 0)
                drain_wait(q_full, (items - 1) & 1, err);
            for (int j = max(0, nk - S::STAGES); j < nk; ++j)
                drain_wait(&k_full[j % S::STAGES], (j / S::STAGES) & 1, err);
            for (int j = max(0, nv - S::STAGES); j < nv; ++j)
                drain_wait(&v_full[j % S::STAGES], (j / S::STAGES) & 1, err);
        } else if (warp < S::ISSUE_WARP + S::CHAINS) {
            // ------------------------------------------------------- products
            constexpr uint32_t idesc_s = make_idesc_f16(128, kKeys, BF16, false);
            const int ksteps = (p.hd + 15) / 16;
            const uint32_t idesc_o = make_idesc_f16(128, ksteps * 16, BF16, true);
            const uint32_t leader = elect_one() ? 1u : 0u;
            const uint32_t aq = smem_u32(sq), ak = smem_u32(sk), av = smem_u32(sv);
            int n = 0, items = 0, listed = 0;
            bool ok = true;
            // S of step g (of the chain's steps), from its K stage.
            auto scores = [&](int g) {
                const int st = g % S::STAGES;
                if (!warp_wait(&k_full[st], (g / S::STAGES) & 1, err, kErrWaitK))
                    return false;
                // One S: the softmax has the last scores in registers.
                if (NC == 1 && g > 0 && !warp_wait(s_free, (g - 1) & 1, err, kErrWaitS))
                    return false;
                tc_fence_after();
                const uint32_t d = tm + (NC == 2 ? (g & 1) * 64 : 0);
#pragma unroll
                for (int k = 0; k < 4 * NC; ++k) {
                    if (k < ksteps) {
                        const uint64_t a = make_smem_desc(aq + (k / 4) * 128 * 128, 16, 1024, kLayoutSW128) + 2 * (k % 4);
                        const uint64_t b = make_smem_desc(ak + st * S::KV_BYTES + (k / 4) * kKeys * 128, 16, 1024, kLayoutSW128) + 2 * (k % 4);
                        umma_ss_if(leader, d, a, b, idesc_s, k > 0 ? 1u : 0u);
                    }
                }
                tc_commit_if(leader, &s_full[NC == 2 ? g & 1 : 0]);
                tc_commit_if(leader, &k_empty[st]);
                return true;
            };
            while (true) {
                const int slot = listed & 1;
                if (!warp_wait(&block_full[slot], (listed >> 1) & 1, err, kErrWaitQ))
                    break;
                const int *from = mine_published + slot * S::BLOCK_INTS;
                const int keys = from[3], sink_steps = from[5], base = from[6], steps = from[7];
                warp_arrive(&block_empty[slot]);
                ++listed;
                if (steps < 0)
                    break;
                if (steps == 0)
                    continue;
                if (!(ok = warp_wait(q_full, items & 1, err, kErrWaitQ)) || !(ok = scores(n)))
                    break;
                if (steps == 1) // every product that reads Q is issued
                    tc_commit_if(leader, q_empty);
                for (int j = 0; j < steps; ++j, ++n) {
                    const int st = n % S::STAGES;
                    if (j + 1 < steps) {
                        if (!(ok = scores(n + 1)))
                            break;
                        if (j + 2 == steps)
                            tc_commit_if(leader, q_empty);
                    }
                    if (!(ok = warp_wait(&v_full[st], (n / S::STAGES) & 1, err, kErrWaitV)))
                        break;
                    const int past = keys - step_key(j, sink_steps, base); // V rows from here on are past the sequence
                    if (past < kKeys) {
                        for (int x = lane; x < NC * (kKeys - past) * 8; x += 32) {
                            const int c = x / ((kKeys - past) * 8), y = x - c * (kKeys - past) * 8;
                            *reinterpret_cast<uint4 *>(sv + st * S::KV_BYTES + c * kKeys * 128 + past * 128 + y * 16) =
                                make_uint4(0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (!(ok = warp_wait(p_full, n & 1, err, kErrWaitP)))
                        break;
                    // The first product overwrites O: the last block's rows have been read.
                    if (j == 0 && items > 0 && !(ok = warp_wait(o_free, (items - 1) & 1, err, kErrWaitO)))
                        break;
                    tc_fence_after();
                    const uint64_t v0 = make_smem_desc(av + st * S::KV_BYTES, kKeys * 128, 1024, kLayoutSW128);
                    const uint32_t a = tm + (NC == 2 ? (n & 1) * 64 : 64);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_ts_if(leader, tm + S::O_COL, a + k * 8, v0 + static_cast<uint64_t>((k * 16 * 128) >> 4), idesc_o,
                                   j > 0 || k > 0 ? 1u : 0u);
                    tc_commit_if(leader, &pv_done[n & 1]);
                    tc_commit_if(leader, &v_empty[st]);
                }
                if (!ok)
                    break;
                ++items;
            }
            tc_commit_if(leader, drain);
            drain_wait(drain, 0, err);
        }
        __syncwarp();
    } else {
        // -------------------------------------------------------------- softmax
        reg_inc<S::SOFT_REGS>();
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = tm + (static_cast<uint32_t>(quarter * 32) << 16);
        const float sl2 = p.scale_log2;
        const int chunks = (p.hd + 15) / 16; // of O, 16 columns each
        int g = 0, listed = 0;
        bool ok = true;
        while (true) {
            const int slot = listed & 1;
            if (!warp_wait(&block_full[slot], (listed >> 1) & 1, err, kErrWaitQ))
                break;
            // What outlives the scores' registers: few values.
            const int *from = mine_published + slot * S::BLOCK_INTS;
            const int t = from[2] + row, pos = from[3] - from[4] + t;
            const int limit = min(from[3], pos + p.right + 1), low = p.window > 0 ? pos - p.window + 1 : 0;
            const int sink_steps = from[5], start = from[6], steps = from[7];
            const bool store = t < from[4];
            const long long base = from[0] * p.o_sb + from[1] * p.o_sh + static_cast<long long>(t) * p.o_st;
            warp_arrive(&block_empty[slot]);
            ++listed;
            if (steps < 0)
                break;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < steps; ++j, ++g) {
                const uint32_t ts = lanes + (NC == 2 ? (g & 1) * 64 : 0);
                if (!(ok = warp_wait(&s_full[NC == 2 ? g & 1 : 0], (NC == 2 ? g >> 1 : g) & 1, err, kErrWaitS)))
                    break;
                tc_fence_after();
                uint32_t raw[kKeys];
                tmem_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
                tmem_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
                tmem_wait_ld();
                if constexpr (NC == 1) { // the next scores may overwrite these
                    tc_fence_before();
                    warp_arrive(s_free);
                }
                float *s = reinterpret_cast<float *>(raw);
                // Columns [0, lo) and [hi, 64) are hidden, save the sinks.  A step wholly
                // before the window shows its sinks alone; one whose hidden start they
                // cover shows all.  A bound is tested only where some row has it.
                const int key = step_key(j, sink_steps, start), sk = p.sinks - key;
                int hi = limit - key, lo = low - key;
                if (lo >= kKeys) {
                    hi = min(hi, sk);
                    lo = 0;
                } else if (sk >= lo) {
                    lo = 0;
                }
                if (__any_sync(0xffffffffu, hi < kKeys)) {
#pragma unroll
                    for (int c = 0; c < kKeys; ++c)
                        if (c >= hi)
                            s[c] = -INFINITY;
                }
                if (__any_sync(0xffffffffu, lo > 0)) {
#pragma unroll
                    for (int c = 0; c < kKeys; ++c)
                        if (c < lo && c >= sk)
                            s[c] = -INFINITY;
                }
                float top[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float *x = s + 16 * q;
                    float v = fmax3(x[0], x[1], x[2]);
#pragma unroll
                    for (int e = 3; e < 15; e += 2)
                        v = fmax3(v, x[e], x[e + 1]);
                    top[q] = fmaxf(v, x[15]);
                }
                const float next = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sl2);
                const bool grow = next > m + 8.0f;
                const float alpha = grow && j > 0 ? ex2_approx(m - next) : 1.f;
                if (grow) {
                    l *= alpha;
                    m = next;
                }
                // A row that has seen no key yet: P = 0, not 2^NaN.
                const float shift = m == -INFINITY ? 0.f : -m;
                float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
                for (int c = 0; c < kKeys / 2; c += 2) {
                    float x0, x1, x2, x3;
                    ffma2(x0, x1, s[2 * c], s[2 * c + 1], sl2, sl2, shift, shift);
                    ffma2(x2, x3, s[2 * c + 2], s[2 * c + 3], sl2, sl2, shift, shift);
                    x0 = ex2_approx(x0);
                    x1 = ex2_approx(x1);
                    x2 = ex2_approx(x2);
                    x3 = ex2_approx(x3);
                    fadd2(a0, a1, a0, a1, x0, x1);
                    fadd2(b0, b1, b0, b1, x2, x3);
                    raw[c] = pack_pair<BF16>(x0, x1);
                    raw[c + 1] = pack_pair<BF16>(x2, x3);
                }
                l += (a0 + a1) + (b0 + b1);
                // The last product is done: its P may be overwritten (one P), O rescaled.
                const bool rescale = j > 0 && __any_sync(0xffffffffu, grow);
                if ((NC == 1 && g > 0) || rescale) {
                    if (!(ok = warp_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, err, kErrWaitO)))
                        break;
                    tc_fence_after();
                }
                if (rescale) {
                    for (int c = 0; c < chunks; ++c) {
                        uint32_t o[16];
                        tmem_ld16(lanes + S::O_COL + c * 16, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st16(lanes + S::O_COL + c * 16, o);
                    }
                }
                __syncwarp();
                tmem_st32(NC == 2 ? ts : lanes + 64, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(p_full);
            }
            if (!ok)
                break;
            const float inv = l > 0.f ? 1.f / l : 0.f;
            if (steps > 0) {
                if (!(ok = warp_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, err, kErrWaitO)))
                    break;
                tc_fence_after();
            }
            for (int c = 0; c < chunks; ++c) {
                uint32_t o[16];
                if (steps > 0) {
                    tmem_ld16(lanes + S::O_COL + c * 16, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[e] = 0u;
                }
                if (c + 1 == chunks && steps > 0) {
                    tc_fence_before();
                    warp_arrive(o_free);
                }
                if (!store)
                    continue;
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    v[e] = __uint_as_float(o[e]) * inv;
                // head_dim is a multiple of 8.
#pragma unroll
                for (int h = 0; h < 16; h += 8) {
                    const int col = c * 16 + h;
                    if (col >= p.hd)
                        continue;
                    if (p.out_dtype == kOutF32) {
                        float *out = static_cast<float *>(p.out) + base + col;
                        if (p.out_vec) {
                            reinterpret_cast<float4 *>(out)[0] = make_float4(v[h], v[h + 1], v[h + 2], v[h + 3]);
                            reinterpret_cast<float4 *>(out)[1] = make_float4(v[h + 4], v[h + 5], v[h + 6], v[h + 7]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                out[e] = v[h + e];
                        }
                    } else {
                        uint16_t *out = static_cast<uint16_t *>(p.out) + base + col;
                        const uint32_t w[4] = {pack_pair<BF16>(v[h], v[h + 1]), pack_pair<BF16>(v[h + 2], v[h + 3]),
                                               pack_pair<BF16>(v[h + 4], v[h + 5]), pack_pair<BF16>(v[h + 6], v[h + 7])};
                        if (p.out_vec) {
                            *reinterpret_cast<uint4 *>(out) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                out[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
                        }
                    }
                }
            }
            __syncwarp();
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::ISSUE_WARP)
        tmem_dealloc(tmem, 512);
}

// (d, token, head, batch) map with boxes of 64 columns x `rows` tokens.
int prompt_map(CUtensorMap *map, const void *base, bool bf16, int hd, int tokens, int heads, int batch,
               const long long *strides, int rows) {
    const uint64_t dims[4] = {static_cast<uint64_t>(hd), static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads),
                              static_cast<uint64_t>(batch)};
    const uint64_t bytes[3] = {static_cast<uint64_t>(strides[2]) * 2, static_cast<uint64_t>(strides[1]) * 2,
                               static_cast<uint64_t>(strides[0]) * 2};
    const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
    return encode_tiled(map, base, bf16, 4, dims, bytes, box, 128);
}

template <int NC, bool BF16> int launch_typed(const PromptParams &p, int sms, cudaStream_t stream) {
    using S = PromptShape<NC>;
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(window_prompt_kernel<NC, BF16>), S::SMEM, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    const long long blocks = static_cast<long long>(p.batch) * p.heads * ((p.q_len + 127) / 128);
    window_prompt_kernel<NC, BF16>
        <<<static_cast<unsigned>(std::min<long long>(blocks, sms)), S::THREADS, S::SMEM, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

} // namespace

int window_prompt_launch(const WindowArgs &a, cudaStream_t stream) {
    PromptParams p{};
    int rc = 0;
    if ((rc = prompt_map(&p.tq, a.q, a.bf16, a.hd, a.q_len, a.heads, a.batch, a.qs, 128)) ||
        (rc = prompt_map(&p.tk, a.k, a.bf16, a.hd, a.kv_len, a.kv_heads, a.batch, a.ks, kKeys)) ||
        (rc = prompt_map(&p.tv, a.v, a.bf16, a.hd, a.kv_len, a.kv_heads, a.batch, a.vs, kKeys)))
        return rc;
    p.out = a.out;
    p.o_sb = a.os[0];
    p.o_sh = a.os[1];
    p.o_st = a.os[2];
    p.lengths = a.lengths;
    p.q_lengths = a.q_lengths;
    p.batch = a.batch;
    p.heads = a.heads;
    p.group = a.heads / a.kv_heads;
    p.q_len = a.q_len;
    p.kv_len = a.kv_len;
    p.hd = a.hd;
    p.window = a.window;
    p.right = a.right;
    p.sinks = a.sinks;
    p.out_dtype = a.out_dtype;
    const int vec = a.out_dtype == kOutF32 ? 4 : 8;
    p.out_vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.os[0] % vec == 0 && a.os[1] % vec == 0 && a.os[2] % vec == 0;
    p.table = (a.lengths || a.q_lengths) && a.batch > 1 && a.batch <= kMaxBatch;
    const double scale = a.scale > 0 ? a.scale : 1.0 / std::sqrt(static_cast<double>(a.hd));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    p.err = a.err;
    const int sms = fmha_sm_count();
    if (a.hd <= 64)
        return a.bf16 ? launch_typed<1, true>(p, sms, stream) : launch_typed<1, false>(p, sms, stream);
    return a.bf16 ? launch_typed<2, true>(p, sms, stream) : launch_typed<2, false>(p, sms, stream);
}

// Query rows that share a key head, up to which the kernel for few rows is taken.
constexpr int kFewRows = 64;

int attention_window(const WindowArgs &a, cudaStream_t stream) {
    if (static_cast<long long>(a.heads / a.kv_heads) * a.q_len <= kFewRows)
        return window_tokens_launch(a, stream);
    return window_prompt_launch(a, stream);
}

} // namespace omni_b200
