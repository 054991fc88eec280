// window_prompt_sm100.cu -- sliding-window attention for prompts and encoders on
// B200 (sm_100a).
//
// softmax(scale * q k^T + mask) v for blocks of 128 query rows.  A window leaves a
// block few keys, so a block is over after some ten steps, and its own chain
// (product, softmax, product) leaves the SM idle between them.  Each CTA therefore
// runs several blocks at once as independent chains, each with queries, keys,
// values, tensor memory and warps of its own: while one waits, another's products and
// exponentials (MUFU: 16 per clock and SM) go on.  Keys come 64 at a time, starting at
// the block's first visible key.
// 8192 tokens, 32/8 heads of 128, window 1024: 167 us, 776 TFLOP/s, with the MUFU 44 % and
// the tensor pipe 43 % busy; 157 us without most products, 149 without exponentials, 122
// without both: the hand-offs between the warps of a chain and the blocks' starts and
// ends bound it.  16 x 16 heads of 64, 1500 tokens, window 257 + 256: 82 us (72 without
// both).  Steps of 128 keys in two chains took 88 us there.
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
// is rarely rescaled.  Steps take turns between two barriers where one side may
// be a step ahead of the other (P written, products done): one barrier's parity would
// mistake the step before the last for the one awaited.
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
constexpr int kBoxBytes = 32 * 64; // a warp's 32 output rows, 64 bytes at a time
constexpr int kMaxBatch = 496; // sequences that the table in shared memory holds

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
    // Barriers by their byte offsets.  k_*, v_*: one per stage; s_full, p_full, pv_done: by
    // the step's parity; block_*: by the block's.  An arrive of each softmax warp: p_full,
    // o_free, s_free; of those and the issuer: block_empty.
    static constexpr uint32_t Q_FULL = 0, Q_EMPTY = 8, K_FULL = 2 * 8, K_EMPTY = 5 * 8, V_FULL = 8 * 8, V_EMPTY = 11 * 8,
                              S_FULL = 14 * 8, PV_DONE = 16 * 8, DRAIN = 18 * 8, P_FULL = 19 * 8, O_FREE = 21 * 8,
                              S_FREE = 22 * 8, BLOCK_FULL = 23 * 8, BLOCK_EMPTY = 25 * 8;
    static_assert(STAGES <= 3, "barrier places");
    static constexpr int BARS = 28, BLOCK_INTS = 12; // per chain; per published block (two of them)
    static constexpr int TABLE_BYTES = (4 * kMaxBatch + 1) * 4; // keys, rows, and (ragged) seq, pre
    static constexpr int BOXES_AT = CHAINS * CHAIN_BYTES, BARS_AT = BOXES_AT + SOFT_WARPS * kBoxBytes;
    static constexpr int TMEM_AT = BARS_AT + CHAINS * BARS * 8, BLOCKS_AT = TMEM_AT + 16;
    static constexpr int TABLE_AT = BLOCKS_AT + CHAINS * 2 * BLOCK_INTS * 4;
    static constexpr int SMEM = TABLE_AT + TABLE_BYTES + 1024;
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};

template <int N> __device__ __forceinline__ void reg_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void reg_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// Shared memory by 32-bit addresses throughout: the scores leave few registers.
// Bounded like mbar_wait; the whole warp goes on or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int *err, int code) {
    bool ok = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok))
        return true;
    const uint64_t start = globaltimer_ns();
    for (uint32_t i = 1; !ok; ++i) {
        ok = mbar_try_wait(bar, parity);
        if (!ok && (i & 127u) == 0) {
            if (*reinterpret_cast<volatile int *>(err) != 0)
                break;
            if (globaltimer_ns() - start > kWaitLimitNs) {
                atomicOr(err, code);
                break;
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}
// Bounded by time only: nothing may be in flight when the CTA ends.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, int *err) {
    const uint64_t start = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (globaltimer_ns() - start > kWaitLimitNs) {
            atomicOr(err, kErrWaitDrain);
            return;
        }
    }
}
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// One arrive per warp, after its lanes.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
        arrive(bar);
}
__device__ __forceinline__ void commit_if(uint32_t issue, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
                 "r"(issue)
                 : "memory");
}
__device__ __forceinline__ void load_4d(uint32_t to, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(to),
                 "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}
__device__ __forceinline__ int get(uint32_t at) {
    int v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint4 get16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void put16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
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

// Keys and queries of sequence b, from the table in shared memory while it has room.
__device__ __forceinline__ int held_keys(const PromptParams &p, const int *table, int b) {
    return p.batch <= kMaxBatch ? table[b] : p.lengths ? max(0, min(p.lengths[b], p.kv_len)) : p.kv_len;
}
__device__ __forceinline__ int held_rows(const PromptParams &p, const int *table, int b) {
    return p.batch <= kMaxBatch ? table[kMaxBatch + b] : p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
}

// Block u of a chain: round k = u / chains goes through the chains forwards and
// backwards in turn.  Blocks of ragged batches come from the table (sequences with
// most keys first, `pre` blocks before each), others with the last rows first, so
// that without a window the longest start first.
__device__ __forceinline__ Block block_at(const PromptParams &p, const int *table, int u, int chains) {
    const int k = u / chains, c = u - k * chains, r = k * chains + ((k & 1) ? chains - 1 - c : c);
    Block it;
    if (p.table) {
        const int *seq = table + 2 * kMaxBatch, *pre = seq + kMaxBatch;
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
    it.n = held_keys(p, table, it.b);
    it.rows = held_rows(p, table, it.b);
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

// Where a chain's tiles, barriers, published blocks and tensor memory lie.  Each
// role builds its own: values that lived from before the roles part would be
// spilled.
template <int NC> struct ChainPlaces {
    using S = PromptShape<NC>;
    uint32_t smem, chain;
    __device__ __forceinline__ ChainPlaces(uint32_t smem, int chain) : smem(smem), chain(chain) {}
    __device__ __forceinline__ uint32_t q() const { return smem + chain * S::CHAIN_BYTES; }
    __device__ __forceinline__ uint32_t k() const { return q() + S::Q_BYTES; }
    __device__ __forceinline__ uint32_t v() const { return k() + S::STAGES * S::KV_BYTES; }
    __device__ __forceinline__ uint32_t bar() const { return smem + S::BARS_AT + chain * (S::BARS * 8); }
    __device__ __forceinline__ uint32_t blocks() const { return smem + S::BLOCKS_AT + chain * (2 * S::BLOCK_INTS * 4); }
    __device__ __forceinline__ uint32_t tmem() const { return get(smem + S::TMEM_AT) + chain * S::COLS; }
};

// A value that the compiler keeps instead of computing it again at each use.
__device__ __forceinline__ uint32_t kept(uint32_t v) {
    asm volatile("" : "+r"(v));
    return v;
}

template <int NC, bool BF16>
__global__ void __launch_bounds__(PromptShape<NC>::THREADS, 1) window_prompt_kernel(const __grid_constant__ PromptParams p) {
    using S = PromptShape<NC>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *all_bars = reinterpret_cast<uint64_t *>(smem + S::BARS_AT);
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(smem + S::TMEM_AT);
    int *table = reinterpret_cast<int *>(smem + S::TABLE_AT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err = p.err;

    if (p.batch <= kMaxBatch) {
        for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
            table[b] = p.lengths ? max(0, min(p.lengths[b], p.kv_len)) : p.kv_len;
            table[kMaxBatch + b] = p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
        }
        __syncthreads();
    }
    if (p.table) {
        int *seq = table + 2 * kMaxBatch, *pre = seq + kMaxBatch;
        for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
            int rank = 0;
            for (int o = 0; o < p.batch; ++o)
                rank += table[o] > table[b] || (table[o] == table[b] && o < b) ? 1 : 0;
            seq[rank] = b;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int sum = 0;
            for (int r = 0; r < p.batch; ++r) {
                pre[r] = sum;
                sum += p.heads * ((table[kMaxBatch + seq[r]] + 127) / 128);
            }
            pre[p.batch] = sum;
        }
    }
    if (threadIdx.x == 0) {
        for (int c = 0; c < S::CHAINS; ++c) {
            uint64_t *bar = all_bars + c * S::BARS;
            for (int i = 0; i < S::BARS; ++i)
                mbar_init(&bar[i], i >= 25 ? 5 : i >= 19 && i < 23 ? 4 : 1);
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

    if (warp >= S::SOFT_WARPS) {
        reg_dec<S::CONTROL_REGS>();
        const ChainPlaces<NC> at(smem_u32(smem), (warp - S::SOFT_WARPS) % S::CHAINS);
        const uint32_t bar = kept(at.bar());
        if (warp < S::ISSUE_WARP) {
            // ------------------------------------------------- blocks and loads
            // Chain c of every CTA before chain c + 1 of any: few blocks spread over the SMs.
            const int chains = gridDim.x * S::CHAINS, mine = static_cast<int>(at.chain) * gridDim.x + blockIdx.x;
            const int listed_blocks = p.table ? table[3 * kMaxBatch + p.batch] : p.batch * p.heads * ((p.q_len + 127) / 128);
            const int blocks = (listed_blocks + chains - 1) / chains * chains; // whole rounds: their last may be empty
            int nk = 0, nv = 0, items = 0, listed = 0;
            bool ok = true;
            auto publish = [&](const Block &it) {
                const int slot = listed & 1;
                if (!warp_wait(bar + S::BLOCK_EMPTY + slot * 8, ((listed >> 1) & 1) ^ 1, err, kErrWaitEmpty))
                    return false;
                if (lane == 0) {
                    const uint32_t to = at.blocks() + slot * (S::BLOCK_INTS * 4);
                    put16(to, it.b, it.h, it.q0, it.n);
                    put16(to + 16, it.rows, it.sink_steps, it.base, it.steps);
                    arrive(bar + S::BLOCK_FULL + slot * 8);
                }
                __syncwarp();
                ++listed;
                return true;
            };
            auto load = [&](uint32_t to, const CUtensorMap *map, uint32_t full, uint32_t empty, int &n, int key, int head, int b) {
                const int st = n % S::STAGES;
                if (!warp_wait(empty + st * 8, ((n / S::STAGES) & 1) ^ 1, err, kErrWaitEmpty))
                    return false;
                if (elect_one()) {
                    arrive_expect_tx(full + st * 8, S::KV_BYTES);
                    for (int c = 0; c < NC; ++c)
                        load_4d(to + st * S::KV_BYTES + c * kKeys * 128, map, full + st * 8, c * 64, key, head, b);
                }
                __syncwarp();
                ++n;
                return true;
            };
            // The first block at or after u (in steps of `chains`) that has rows.
            auto find = [&](int &u, Block &it) {
                for (; u < blocks; u += chains) {
                    it = block_at(p, table, u, chains);
                    if (!it.skip)
                        return true;
                }
                return false;
            };
            int u = mine;
            Block it;
            bool more = find(u, it);
            ok = !more || publish(it);
            while (ok && more) {
                const int head = it.h / p.group;
                if (it.steps > 0) {
                    if (!(ok = warp_wait(bar + S::Q_EMPTY, (items & 1) ^ 1, err, kErrWaitEmpty)))
                        break;
                    if (elect_one()) {
                        arrive_expect_tx(bar + S::Q_FULL, S::Q_BYTES);
                        for (int c = 0; c < NC; ++c)
                            load_4d(at.q() + c * 128 * 128, &p.tq, bar + S::Q_FULL, c * 64, it.q0, it.h, it.b);
                    }
                    __syncwarp();
                    ++items;
                    // Keys a step ahead of values: they are wanted a step earlier.
                    if (!(ok = load(at.k(), &p.tk, bar + S::K_FULL, bar + S::K_EMPTY, nk, step_key(0, it.sink_steps, it.base), head, it.b)))
                        break;
                }
                // The next block is found while this one's loads are under way.  (Bringing its
                // queries to L2 here cost more than it saved: 203 against 167 us.)
                const int look = it.steps > 1 ? 1 : 0;
                Block next;
                for (int j = 0; ok && (j < it.steps || j == look); ++j) {
                    if (j + 1 < it.steps)
                        ok = load(at.k(), &p.tk, bar + S::K_FULL, bar + S::K_EMPTY, nk, step_key(j + 1, it.sink_steps, it.base), head, it.b);
                    if (ok && j < it.steps)
                        ok = load(at.v(), &p.tv, bar + S::V_FULL, bar + S::V_EMPTY, nv, step_key(j, it.sink_steps, it.base), head, it.b);
                    if (!ok || j != look)
                        continue;
                    u += chains;
                    more = find(u, next);
                    if (!more)
                        continue;
                    ok = publish(next);
                }
                it = next;
            }
            if (ok) {
                Block end{};
                end.steps = -1;
                publish(end);
            }
            // Every copy lands before the CTA ends.
            if (items > 0)
                drain_wait(bar + S::Q_FULL, (items - 1) & 1, err);
            for (int j = max(0, nk - S::STAGES); j < nk; ++j)
                drain_wait(bar + S::K_FULL + j % S::STAGES * 8, (j / S::STAGES) & 1, err);
            for (int j = max(0, nv - S::STAGES); j < nv; ++j)
                drain_wait(bar + S::V_FULL + j % S::STAGES * 8, (j / S::STAGES) & 1, err);
        } else if (warp < S::ISSUE_WARP + S::CHAINS) {
            // ------------------------------------------------------- products
            constexpr uint32_t idesc_s = make_idesc_f16(128, kKeys, BF16, false);
            const int ksteps = (p.hd + 15) / 16;
            const uint32_t idesc_o = make_idesc_f16(128, ksteps * 16, BF16, true);
            const uint32_t leader = elect_one() ? 1u : 0u;
            const uint32_t tm = kept(at.tmem());
            const uint64_t dq = make_smem_desc(at.q(), 16, 1024, kLayoutSW128);
            const uint64_t dk = make_smem_desc(at.k(), 16, 1024, kLayoutSW128);
            const uint64_t dv = make_smem_desc(at.v(), kKeys * 128, 1024, kLayoutSW128);
            int n = 0, items = 0, listed = 0;
            bool ok = true;
            // S of step g (of the chain's steps), from its K stage.
            auto scores = [&](int g) {
                const int st = g % S::STAGES;
                if (!warp_wait(bar + S::K_FULL + st * 8, (g / S::STAGES) & 1, err, kErrWaitK))
                    return false;
                // One S: the softmax has the last scores in registers.
                if (NC == 1 && g > 0 && !warp_wait(bar + S::S_FREE, (g - 1) & 1, err, kErrWaitS))
                    return false;
                tc_fence_after();
                const uint32_t d = tm + (NC == 2 ? (g & 1) * 64 : 0);
                const uint64_t b = dk + static_cast<uint64_t>(st * (S::KV_BYTES >> 4));
#pragma unroll
                for (int k = 0; k < 4 * NC; ++k)
                    if (k < ksteps)
                        umma_ss_if(leader, d, dq + (k / 4) * (128 * 128 >> 4) + 2 * (k % 4),
                                   b + (k / 4) * (kKeys * 128 >> 4) + 2 * (k % 4), idesc_s, k > 0 ? 1u : 0u);
                commit_if(leader, bar + S::S_FULL + (NC == 2 ? (g & 1) * 8 : 0));
                commit_if(leader, bar + S::K_EMPTY + st * 8);
                return true;
            };
            while (true) {
                const int slot = listed & 1;
                if (!warp_wait(bar + S::BLOCK_FULL + slot * 8, (listed >> 1) & 1, err, kErrWaitQ))
                    break;
                const uint32_t from = at.blocks() + slot * (S::BLOCK_INTS * 4);
                const int keys = get(from + 12), sink_steps = get(from + 20), base = get(from + 24), steps = get(from + 28);
                warp_arrive(bar + S::BLOCK_EMPTY + slot * 8);
                ++listed;
                if (steps < 0)
                    break;
                if (steps == 0)
                    continue;
                if (!(ok = warp_wait(bar + S::Q_FULL, items & 1, err, kErrWaitQ)) || !(ok = scores(n)))
                    break;
                if (steps == 1) // every product that reads Q is issued
                    commit_if(leader, bar + S::Q_EMPTY);
                for (int j = 0; j < steps; ++j, ++n) {
                    const int st = n % S::STAGES;
                    if (j + 1 < steps) {
                        if (!(ok = scores(n + 1)))
                            break;
                        if (j + 2 == steps)
                            commit_if(leader, bar + S::Q_EMPTY);
                    }
                    if (!(ok = warp_wait(bar + S::V_FULL + st * 8, (n / S::STAGES) & 1, err, kErrWaitV)))
                        break;
                    const int past = keys - step_key(j, sink_steps, base); // V rows from here on are past the sequence
                    if (past < kKeys) {
                        for (int x = lane; x < NC * (kKeys - past) * 8; x += 32) {
                            const int c = x / ((kKeys - past) * 8), y = x - c * (kKeys - past) * 8;
                            put16(at.v() + st * S::KV_BYTES + c * kKeys * 128 + past * 128 + y * 16, 0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (!(ok = warp_wait(bar + S::P_FULL + (n & 1) * 8, (n >> 1) & 1, err, kErrWaitP)))
                        break;
                    // The first product overwrites O: the last block's rows have been read.
                    if (j == 0 && items > 0 && !(ok = warp_wait(bar + S::O_FREE, (items - 1) & 1, err, kErrWaitO)))
                        break;
                    tc_fence_after();
                    const uint64_t v0 = dv + static_cast<uint64_t>(st * (S::KV_BYTES >> 4));
                    const uint32_t a = tm + (NC == 2 ? (n & 1) * 64 : 64);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_ts_if(leader, tm + S::O_COL, a + k * 8, v0 + static_cast<uint64_t>((k * 16 * 128) >> 4), idesc_o,
                                   j > 0 || k > 0 ? 1u : 0u);
                    commit_if(leader, bar + S::PV_DONE + (n & 1) * 8);
                    commit_if(leader, bar + S::V_EMPTY + st * 8);
                }
                if (!ok)
                    break;
                ++items;
            }
            commit_if(leader, bar + S::DRAIN);
            drain_wait(bar + S::DRAIN, 0, err);
        }
        __syncwarp();
    } else {
        // -------------------------------------------------------------- softmax
        reg_inc<S::SOFT_REGS>();
        const ChainPlaces<NC> at(smem_u32(smem), warp / 4);
        const uint32_t bar = kept(at.bar());
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = kept(at.tmem() + (static_cast<uint32_t>(quarter * 32) << 16));
        const float sl2 = p.scale_log2;
        const int chunks = (p.hd + 15) / 16; // of O, 16 columns each
        const uint32_t box = kept(at.smem + S::BOXES_AT + warp * kBoxBytes);
        int g = 0, listed = 0;
        bool ok = true;
        while (true) {
            const int slot = listed & 1;
            if (!warp_wait(bar + S::BLOCK_FULL + slot * 8, (listed >> 1) & 1, err, kErrWaitQ))
                break;
            // What outlives the scores' registers: few values.
            const uint32_t from = at.blocks() + slot * (S::BLOCK_INTS * 4);
            const uint4 who = get16(from), what = get16(from + 16);
            const int t = static_cast<int>(who.z) + row, keys = who.w, pos = keys - static_cast<int>(what.x) + t;
            const int limit = min(keys, pos + p.right + 1), low = p.window > 0 ? pos - p.window + 1 : 0;
            const int sink_steps = what.y, start = what.z, steps = what.w;
            const int left = static_cast<int>(what.x) - static_cast<int>(who.z) - quarter * 32; // rows of this warp that exist
            const long long base = static_cast<int>(who.x) * p.o_sb + static_cast<int>(who.y) * p.o_sh +
                                   static_cast<long long>(t - lane) * p.o_st;
            warp_arrive(bar + S::BLOCK_EMPTY + slot * 8);
            ++listed;
            if (steps < 0)
                break;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < steps; ++j, ++g) {
                const uint32_t ts = lanes + (NC == 2 ? (g & 1) * 64 : 0);
                if (!(ok = warp_wait(bar + S::S_FULL + (NC == 2 ? (g & 1) * 8 : 0), (NC == 2 ? g >> 1 : g) & 1, err, kErrWaitS)))
                    break;
                tc_fence_after();
                uint32_t raw[kKeys];
                tmem_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
                tmem_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
                tmem_wait_ld();
                if constexpr (NC == 1) { // the next scores may overwrite these
                    tc_fence_before();
                    warp_arrive(bar + S::S_FREE);
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
                    // To the type of v, as the tensor cores take them: up to half a step of each
                    // (8192 tokens in bf16: off by 0.0022, relative, where fp32 weights give
                    // 0.0016; fp16 2.7e-5 and 1.9e-5).  l is the sum of the unrounded values.
                    raw[c] = pack_pair<BF16>(x0, x1);
                    raw[c + 1] = pack_pair<BF16>(x2, x3);
                }
                l += (a0 + a1) + (b0 + b1);
                // The last product is done: its P may be overwritten (one P), O rescaled.
                const bool rescale = j > 0 && __any_sync(0xffffffffu, grow);
                if ((NC == 1 && g > 0) || rescale) {
                    if (!(ok = warp_wait(bar + S::PV_DONE + ((g - 1) & 1) * 8, ((g - 1) >> 1) & 1, err, kErrWaitO)))
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
                warp_arrive(bar + S::P_FULL + (g & 1) * 8);
            }
            if (!ok)
                break;
            // Zeros for a row that sees no key, which `limit` tells; a sum that is no positive
            // number otherwise stands for scores that are not finite, and gives NaN.
            const float inv = limit > 0 ? 1.f / l : 0.f;
            if (steps > 0) {
                if (!(ok = warp_wait(bar + S::PV_DONE + ((g - 1) & 1) * 8, ((g - 1) >> 1) & 1, err, kErrWaitO)))
                    break;
                tc_fence_after();
            }
            // 64 bytes of each of the warp's rows at a time, through shared memory: a lane
            // has a row, but the stores take four lanes to a row and write whole sectors.
            const int size = p.out_dtype == kOutF32 ? 4 : 2, width = 64 / size;
            for (int c = 0; c < p.hd; c += width) {
                uint32_t w[16];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1 && size == 4)
                        break;
                    uint32_t o[16];
                    // Columns past head_dim in a 32-column pass: not written below.
                    if (steps > 0 && c + 16 * h < p.hd) {
                        tmem_ld16(lanes + S::O_COL + c + 16 * h, o);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
                    if (size == 4) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            w[e] = o[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            w[8 * h + e] = pack_pair<BF16>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                    }
                }
                if (c + width >= p.hd && steps > 0) { // O may be overwritten
                    tc_fence_before();
                    warp_arrive(bar + S::O_FREE);
                }
                __syncwarp(); // the last pass's box has been read
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    put16(box + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = k * 8 + lane / 4, j = lane & 3, col = c + j * (width / 4);
                    if (r >= left || col >= p.hd)
                        continue;
                    const uint4 v = get16(box + r * 64 + ((j ^ ((r >> 1) & 3)) << 4));
                    const long long place = base + r * p.o_st + col;
                    if (p.out_vec) {
                        *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.out) + place * size) = v;
                    } else if (size == 4) {
                        uint32_t *out = static_cast<uint32_t *>(p.out) + place;
                        out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
                    } else {
                        uint16_t *out = static_cast<uint16_t *>(p.out) + place;
                        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            out[e] = static_cast<uint16_t>(x[e / 2] >> (16 * (e & 1)));
                    }
                }
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == S::ISSUE_WARP)
        tmem_dealloc(*tmem_holder, 512);
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

// The cheaper kernel, in tenths of a microsecond as measured.  Few rows: the keys
// that every 16 rows read, and at least one warp's share of them; prompts: a block's
// steps one after another, in rounds of what the chains of the SMs hold.  Measured,
// prompts / few rows: 16 x 8/2 heads of 128, window 1024, 16 queries 21.1 / 21.3 us,
// 32 queries 20.9 / 28.0; one sequence, 16384 keys, 8/1 heads, 64 queries 186 / 43;
// 4 x 8 heads of 64, 4096 keys, 128 queries 58 / 52, 256 queries 58 / 101.
int attention_window(const WindowArgs &a, cudaStream_t stream) {
    const double around = a.window > 0 ? static_cast<double>(a.window) + a.right + a.sinks : a.kv_len;
    const double few_keys = std::min<double>(a.kv_len, around + a.q_len);
    const long long tiles = (static_cast<long long>(a.heads / a.kv_heads) * a.q_len + 15) / 16;
    const double read = few_keys * tiles * a.batch * a.kv_heads * a.hd / 155000.0;
    const double share = few_keys / 64 / window_tokens_parts(a) * 7;
    const double few_cost = 75 + std::max(read, share);
    const double steps = std::min<double>(a.kv_len, around + 127) / kKeys + 1;
    const double blocks = static_cast<double>(a.batch) * a.heads * ((a.q_len + 127) / 128);
    const double prompt_cost = 70 + 7 * steps * std::max(1.0, blocks / (1.45 * fmha_sm_count()));
    if (tiles <= 65535 && few_cost <= prompt_cost)
        return window_tokens_launch(a, stream);
    return window_prompt_launch(a, stream);
}

} // namespace omni_b200
