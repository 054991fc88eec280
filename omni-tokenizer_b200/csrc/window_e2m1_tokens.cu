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
// exact in f16, P <= 2^15 is rounded to 11 bits there (bf16: 8), and a bf16 row of q is
// multiplied by the power of two that brings its largest element to [2^14, 2^15): elements
// down to 2^-28 of it keep all their bits, what is below loses less than 2^-39 of it.
//
// The bound is the cache's bytes.  A block of 16 tokens of a head (2304 bytes at 128 columns)
// is one contiguous piece; each warp copies its own blocks, two at a time, to a ring in shared
// memory (a bulk copy for a block, no barrier between warps) and keeps its own softmax state.
// Converting takes a conversion and a product for two elements, 128 instructions of a block's
// 248; the rest is kept short: a lane looks up the pages of 32 blocks at once, and the running maximum
// is lazy (other lanes are asked only when some weight would be above 2^15).
// 16 sequences of 65536 keys, 32/8 heads of 128: 198 us, 6.09 TB/s (copies alone 185, products
// alone 176); 64 of up to 16384: 123 us, and 133 to 136 in a long run at the 1.81 GHz that the
// power cap leaves.  248 instructions for a block of 16 tokens, issue slots 59 % busy, ALU 47 %.
//
// Two ways to split the keys over CTAs:
//   * few tiles of rows: a cluster takes each; its parts meet in distributed shared memory, in
//     rank order (no atomics, no workspace, one launch);
//   * else the blocks of all tiles, one list, go to CTAs that are all on the GPU at once, the
//     same number to each whatever the sequences' lengths are.  A tile that is one CTA's is
//     finished there; parts of others go to the workspace, and a second kernel joins them.
#include "cache_e2m1.cuh"
#include "fmha.h"
#include "layer.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace omni_b200 {
namespace {

constexpr int kMaxParts = 16;
constexpr int kMostRows = 512; // of a key head, group * q_len
// A row's largest key so far has the weight 2^kTop (log2 units, as scores), and a score may be
// kLazy above it before the reference follows: weights reach 2^15 of f16's 2^16, and at the other
// end lose at most 2^-25 / 2^kTop = 2^-32 of the largest each.
constexpr float kTop = 7.f, kLazy = 8.f;

struct TokensParams {
    CacheView cache;
    const uint16_t *q;
    void *out;
    float *parts_at; // of the list's parts: [CTA][first or last tile][m, l of the rows, then rows x D]
    long long qs[3], os[3];
    const int *lengths, *q_lengths;
    int parts; // CTAs of a cluster, or 0: the list
    int ctas;  // of the list
    uint32_t group_inv; // ceil(2^20 / group): exact for quotients of numbers up to kMostRows by group up to it
    int batch, kv_heads, group, q_len, kv_len, hd, tiles; // tiles of rows that a sequence may have
    int window, right, sinks;
    int out_dtype;
    float scale_log2;
    int *err;
};

// CTAs on an SM, by registers; shared memory allows no more of 24 rows either (90 KB at 128
// columns).  Some instances spill all the same, bytes stored and loaded: at 128 columns the list
// 28 and 32 with 8 rows, 108 and 120 with 24, the f16 cluster of 24 rows 18 and 24; at 96 the list
// of 8 rows up to 12 and 48.  (More for narrow heads do not help eight rows: 64 x up to 16384
// keys of 64, 81 us with four, 82 with five; 16 rows of 64 columns 134 with two, 119 with three.)
constexpr int ctas_of_sm(int width, int rows) { return rows == 8 ? 4 : rows == 16 && width <= 64 ? 3 : 2; }

template <int D, int NT> struct TokensShape {
    static constexpr int BLOCK = CacheBlock<D>::BYTES;
    static constexpr int WARPS = 4, CTAS = ctas_of_sm(D, 8 * NT);
    static constexpr int STAGES = 2, STAGE = 2 * BLOCK; // a pair that is read, one on its way
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int ROWS = 8 * NT;
    // The warps' results: m, l of each and of the CTA, outputs.
    static constexpr int PARTS = (2 * WARPS + 2) * ROWS * 4 + WARPS * ROWS * (D + 4) * 4;
    static constexpr int SMEM = RING + PARTS;
    static constexpr int SLOT = ROWS * (D + 2); // floats of a part in the workspace
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with zeros to add to.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// One contiguous piece (16-byte addresses and size) to shared memory, counted by `bar`.
__device__ __forceinline__ void copy_piece(uint32_t to, unsigned long long from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
                 "r"(bytes), "r"(bar)
                 : "memory");
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

// A tile of rows of a sequence and key head, and the blocks of the cache that it sees: [0,
// sink_blocks) and from `begin` on, in that order `blocks` of them.
struct Tile {
    int n, m, row0, rows, pos0;
    int first, last, low, high, sink, sink_blocks, begin, blocks;
};
__device__ __forceinline__ int query_of(const TokensParams &p, int row) { return static_cast<int>(row * p.group_inv >> 20); }
__device__ __forceinline__ void lengths_of(const TokensParams &p, int b, int &n, int &m) {
    n = max(0, min(p.lengths[b], p.kv_len));
    m = p.q_lengths ? max(0, min(p.q_lengths[b], p.q_len)) : p.q_len;
}
template <int ROWS> __device__ __forceinline__ Tile tile_of(const TokensParams &p, int n, int m, int tile) {
    Tile t;
    t.n = n;
    t.m = m;
    // Rows r of the tile: query (row0 + r) / group, head kvh * group + (row0 + r) % group.
    t.row0 = tile * ROWS;
    t.rows = min(ROWS, p.group * m - t.row0);
    t.pos0 = n - m;
    // Keys that some row of the tile sees: [0, sink) and [low, high).
    t.first = t.pos0 + query_of(p, t.row0);
    t.last = t.pos0 + query_of(p, t.row0 + max(t.rows, 1) - 1);
    t.high = t.rows > 0 ? max(0, min(n, t.last + p.right + 1)) : 0;
    t.low = p.window > 0 ? max(0, min(t.first - p.window + 1, t.high)) : 0;
    t.sink = min(p.sinks, t.low);
    t.sink_blocks = (t.sink + kCacheBlock - 1) / kCacheBlock;
    t.begin = max(t.low / kCacheBlock, t.sink_blocks);
    t.blocks = t.sink_blocks + max(0, (t.high + kCacheBlock - 1) / kCacheBlock - t.begin);
    return t;
}
// Its length in the list: beginning and ending a tile takes a CTA as long as some blocks do
// (3 us against 0.22 us for one; 64 x up to 16384 keys 124 us with 8 here, 122 with 16), so it counts for those as well.
constexpr int kTileCost = 16;
__device__ __forceinline__ int listed(const Tile &t) { return t.rows > 0 ? kTileCost + t.blocks : 0; }
// Blocks of all tiles of a sequence's key head: 2^31 and more of them where 32 tiles see 2^30 keys.
template <int ROWS> __device__ __forceinline__ long long listed_of(const TokensParams &p, int b) {
    int n, m;
    long long sum = 0;
    lengths_of(p, b, n, m);
    for (int i = 0; i < p.tiles; ++i)
        sum += listed(tile_of<ROWS>(p, n, m, i));
    return sum;
}

__device__ __forceinline__ void store_out(const TokensParams &p, const Tile &t, int b, int kvh, int r, int col, float v, float l) {
    const int row = t.row0 + r, query = query_of(p, row);
    // Zeros for a row that sees no key, which its position tells: a sum that is no positive
    // number otherwise stands for scores that are not finite, and gives NaN.
    v = min(t.n, t.pos0 + query + p.right + 1) > 0 ? v / l : 0.f;
    const long long to = b * p.os[0] + (kvh * p.group + row - query * p.group) * p.os[1] + query * p.os[2] + col;
    if (p.out_dtype == kOutF32)
        static_cast<float *>(p.out)[to] = v;
    else if (p.out_dtype == kOutBF16)
        static_cast<__nv_bfloat16 *>(p.out)[to] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p.out)[to] = __float2half_rn(v);
}

// What a CTA does at a time: pairs of blocks j0, j0 + step, ... below j1 of a tile.  slot: where
// its part goes in the workspace, or -1: it is the whole tile.
struct Segment {
    Tile tile;
    int b, kvh, j0, j1, slot;
    __device__ __forceinline__ int block_of(int i) const { return i < tile.sink_blocks ? i : tile.begin + i - tile.sink_blocks; }
};

// The warps' results in shared memory.
template <int D, int NT> struct Parts {
    using S = TokensShape<D, NT>;
    float m[S::WARPS][S::ROWS];
    union {
        float l[S::WARPS][S::ROWS];
        uint32_t lost[S::WARPS][S::ROWS]; // before: groups of columns that are NaN, a bit for each
    };
    float cta_m[S::ROWS], cta_l[S::ROWS];
    float o[S::WARPS][S::ROWS][D + 4];
};

template <int D, int NT, bool BF16> struct Worker {
    using S = TokensShape<D, NT>;
    using B = CacheBlock<D>;
    using C = Columns<D>;
    static constexpr int ROWS = S::ROWS, ST = S::STAGES, W = S::WARPS;
    static_assert(sizeof(Parts<D, NT>) == S::PARTS, "the parts' place");

    const TokensParams &p;
    const int step, warp, lane;
    const uint32_t ring;
    uint64_t *const full; // a stage's two copies have landed
    // Where the warp is in its ring: the stage of the next pair, and the parity of its barrier.
    int stage_at = 0;
    uint32_t parity = 0;
    // Of the segment that is fetched: pairs [whole0, whole1) every row sees whole, so they need no
    // mask (sinks are left to it, and so is everything once a page is none of the cache's).
    int whole0 = 0, whole1 = 0, pairs = 0;
    // Lane l knows where block l % 2 of pair k + l / 2 is, k a multiple of 16 (0: nowhere), and
    // copies it; and the pages of the next 16 pairs, or of the next segment's first.
    unsigned long long place = 0;
    int page_next = 0, within_next = 0, page_then = 0, within_then = 0;

    __device__ __forceinline__ Worker(const TokensParams &p_, int step_, uint8_t *smem, uint64_t *bars)
        : p(p_), step(step_), warp(threadIdx.x >> 5), lane(threadIdx.x & 31),
          ring(smem_u32(smem) + (threadIdx.x >> 5) * ST * S::STAGE), full(bars + (threadIdx.x >> 5) * ST) {}

    __device__ __forceinline__ void next_stage() {
        stage_at ^= 1;
        parity ^= stage_at ^ 1;
    }
    __device__ __forceinline__ int page_at(const Segment &s, int k, int &within) const {
        const int i = s.j0 + (warp + (k + (lane >> 1)) * W) * step + (lane & 1);
        return i < s.j1 ? p.cache.page_of(s.b, s.block_of(i), within) : -2;
    }
    __device__ __forceinline__ void copy(const Segment &s, int k, int stage, int &whole1) {
        if ((k & 15) == 0) {
            if (__any_sync(0xffffffffu, page_next == -1))
                whole1 = -1;
            place = page_next >= 0 ? reinterpret_cast<unsigned long long>(p.cache.block_at(page_next, s.kvh, within_next, S::BLOCK)) : 0ull;
            page_next = page_at(s, k + 16, within_next);
        }
        if ((lane >> 1) == (k & 15)) {
            mbar_arrive_expect_tx(full + stage, place ? S::BLOCK : 0);
            if (place)
                copy_piece(ring + stage * S::STAGE + (lane & 1) * S::BLOCK, place, S::BLOCK, smem_u32(full + stage));
        }
    }
    // Asks for the pages of a segment's first pairs, and begins it: its first pair to `stage`.
    __device__ __forceinline__ void ask(const Segment &s) { page_then = page_at(s, 0, within_then); }
    __device__ __forceinline__ void begin(const Segment &s, int stage) {
        const Tile &tile = s.tile;
        const int limit_all = min(tile.n, tile.first + p.right + 1), floor_all = p.window > 0 ? tile.last - p.window + 1 : 0;
        const int ahead = tile.sink_blocks - tile.begin;
        whole0 = max(tile.sink_blocks, (max(floor_all, 0) + kCacheBlock - 1) / kCacheBlock + ahead);
        whole1 = min(s.j1, max(limit_all, 0) / kCacheBlock + ahead) - 1;
        const int mine = s.j1 - s.j0 - warp * step;
        pairs = mine > 0 ? (mine + W * step - 1) / (W * step) : 0;
        page_next = page_then;
        within_next = within_then;
        if (pairs)
            copy(s, 0, stage, whole1);
    }

    // Its rows of q, as they are: this lane's columns of rows g.
    uint4 queries[NT][C::WORDS];
    __device__ __forceinline__ void load_queries(const Segment &s) {
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = s.tile.row0 + 8 * t + g, query = query_of(p, r);
            const bool real = 8 * t + g < s.tile.rows;
            const uint16_t *q = p.q + s.b * p.qs[0] + (s.kvh * p.group + r - query * p.group) * p.qs[1] + query * p.qs[2];
#pragma unroll
            for (int j = 0; j < C::WORDS; ++j) {
                const int col = C::first(j, c);
                queries[t][j] = real && col < p.hd ? *reinterpret_cast<const uint4 *>(q + col) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    }

    // The softmax of the segment that has begun, the warp's share of it, to `parts`; begins the
    // next one (NULL: there is none) before the last pair's turn.
    __device__ __forceinline__ void attend(const Segment &seg, const Segment *next, Parts<D, NT> &parts) {
        const int whole0 = this->whole0, pairs = this->pairs;
        int whole1 = this->whole1;
        if (next)
            ask(*next);
        const Tile &tile = seg.tile;
        const int g = lane >> 2, c = lane & 3, j1 = seg.j1;
        // The queries as B operands, and the masks of columns 2c and 2c + 1.
        uint32_t qb[NT][D / 16][2];
        float factor[NT][2]; // from S to log2 units
        int limit[NT][2], floor_[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint4 (&w)[C::WORDS] = queries[t];
            uint32_t top2 = 0;
#pragma unroll
            for (int j = 0; j < C::WORDS; ++j) {
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
                const int col = 8 * t + 2 * c + h, pos = tile.pos0 + query_of(p, tile.row0 + col);
                const int of_col = __shfl_sync(0xffffffffu, exponent, 4 * (2 * c + h));
                // Not 0, so that a hidden key's -inf stays -inf.
                factor[t][h] = fmaxf(p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - of_col) << 23), 1.4e-45f);
                limit[t][h] = col < tile.rows ? min(tile.n, pos + p.right + 1) : tile.n; // a row that is none: anything finite
                floor_[t][h] = col < tile.rows && p.window > 0 ? pos - p.window + 1 : 0;
            }
        }

        float o[NT][D / 16][4];
        float ref[NT][2], sum[NT][2], bar[NT][2]; // bar: what a score of S must not be above
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
                o[t][x][0] = o[t][x][1] = o[t][x][2] = o[t][x][3] = 0.f;
            ref[t][0] = ref[t][1] = 0.f;
            bar[t][0] = bar[t][1] = -INFINITY;
            sum[t][0] = sum[t][1] = 0.f;
        }
        bool none[NT][2]; // no score yet
#pragma unroll
        for (int t = 0; t < NT; ++t)
            none[t][0] = none[t][1] = true;

        bool lost = false; // parts.lost holds what the masked pairs noted
        // One pair, at `at` in the ring.  (Two instances, so that pairs without a mask carry none of its instructions.)
        auto attend_pair = [&](auto masked, uint32_t at, int i0) {
            constexpr bool MASKED = decltype(masked)::value;
            int key0 = 0, key1 = 0;
            uint32_t bad = 0; // blocks whose page is none
            if constexpr (MASKED) {
                int within;
                bad = (p.cache.page_of(seg.b, seg.block_of(i0), within) < 0 ? 1u : 0u) |
                      (i0 + 1 < j1 && p.cache.page_of(seg.b, seg.block_of(i0 + 1), within) < 0 ? 2u : 0u);
                key0 = seg.block_of(i0) * kCacheBlock;
                key1 = i0 + 1 < j1 ? seg.block_of(i0 + 1) * kCacheBlock : tile.n; // no token is there
                // Values that no row sees may be anything: their scales become zeros.  So do those that
                // are not finite where the rows see different keys (0 * NaN would reach the others),
                // and the rows that see one are noted: they get their NaN in the end.
                const int u = lane / kCacheBlock, r = lane % kCacheBlock, token = (u ? key1 : key0) + r;
                const bool unseen = (bad >> u & 1u) || token >= tile.high || (token < tile.low && token >= tile.sink);
                uint32_t groups = 0;
#pragma unroll
                for (int group = 0; group < B::G; ++group) {
                    const uint32_t scale_at = at + u * S::BLOCK + B::VALUE_SCALES + 2 * B::value_scale(r, group);
                    bool clear = unseen;
                    if (tile.first != tile.last && !unseen) {
                        uint16_t scale;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(scale) : "r"(scale_at) : "memory");
                        clear = not_finite(scale);
                        groups |= clear ? 1u << group : 0u;
                    }
                    if (clear)
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(scale_at), "h"(static_cast<uint16_t>(0)) : "memory");
                }
                if (__any_sync(0xffffffffu, groups)) {
                    if (!lost && lane < ROWS)
                        parts.lost[warp][lane] = 0;
                    lost = true;
                    __syncwarp();
                    for (int row = 0; groups && row < tile.rows; ++row) {
                        const int pos = tile.pos0 + query_of(p, tile.row0 + row);
                        if (token <= pos + p.right && (p.window <= 0 || token > pos - p.window || token < p.sinks))
                            atomicOr(&parts.lost[warp][row], groups);
                    }
                }
                fence_proxy_async_smem(); // the next copy's writes come after these
                __syncwarp();
            }
            // S^T: tokens g (rows 0 to 7) and g + 8 of each block; the blocks' products take turns,
            // so that none waits for the one before it.
            float s[2][NT][4];
            uint32_t kw[2][2][C::WORDS], scales[2][C::TOGETHER ? 1 : C::WORDS];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t row = at + u * S::BLOCK + B::KEYS + (g + 8 * h) * (D / 2);
                    if constexpr (C::TOGETHER)
                        shared_words<C::WORDS>(row + c * 4 * C::WORDS, kw[u][h]);
                    else
#pragma unroll
                        for (int j = 0; j < C::WORDS; ++j)
                            shared_words<1>(row + j * 16 + c * 4, &kw[u][h][j]);
                }
#pragma unroll
                for (int j = 0; j < (C::TOGETHER ? 1 : C::WORDS); ++j) // both tokens' scales of the lane's group
                    shared_words<1>(at + u * S::BLOCK + B::KEY_SCALES + 2 * B::key_scale(g, C::first(j, c) / 32), &scales[u][j]);
            }
#pragma unroll
            for (int j = 0; j < C::WORDS; ++j) {
                uint32_t a[2][2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t both = scales[u][C::TOGETHER ? 0 : j];
                    const uint32_t s_g = __byte_perm(both, 0, 0x1010), s_g8 = __byte_perm(both, 0, 0x3232);
                    uint32_t x[4], y[4];
                    f16x8(kw[u][0][j], x);
                    f16x8(kw[u][1][j], y);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        a[u][e][0] = hmul2(x[2 * e], s_g);
                        a[u][e][1] = hmul2(y[2 * e], s_g8);
                        a[u][e][2] = hmul2(x[2 * e + 1], s_g);
                        a[u][e][3] = hmul2(y[2 * e + 1], s_g8);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (j == 0 && e == 0)
                                mma16816_first(s[u][t], a[u][e], qb[t][2 * j + e][0], qb[t][2 * j + e][1]);
                            else
                                mma16816(s[u][t], a[u][e], qb[t][2 * j + e][0], qb[t][2 * j + e][1]);
            }
            if constexpr (MASKED) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) { // token g + 8 (e / 2), query 2c + e % 2
                            const int token = (u ? key1 : key0) + g + 8 * (e >> 1);
                            const bool seen = token < limit[t][e & 1] && (token >= floor_[t][e & 1] || token < p.sinks);
                            s[u][t][e] = seen ? (bad >> u & 1u ? NAN : s[u][t][e]) : -INFINITY;
                        }
            }
            bool above = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    above |= fmaxf(fmax3(s[0][t][h], s[0][t][h + 2], s[1][t][h]), s[1][t][h + 2]) > bar[t][h];
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float times[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float top = fmaxf(fmax3(s[0][t][h], s[0][t][h + 2], s[1][t][h]), s[1][t][h + 2]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        times[h] = 1.f;
                        const float next = fmaf(top, factor[t][h], -kTop);
                        if (top > bar[t][h] || (!none[t][h] && next > ref[t][h])) {
                            times[h] = none[t][h] ? 0.f : ex2_approx(ref[t][h] - next);
                            none[t][h] = false;
                            ref[t][h] = next;
                            bar[t][h] = (next + (kTop + kLazy)) / factor[t][h];
                        }
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
            uint32_t pb[2][NT][2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[u][t][e] = ex2_approx(fmaf(s[u][t][e], factor[t][e & 1], -ref[t][e & 1]));
                        sum[t][e & 1] += s[u][t][e];
                    }
                    pb[u][t][0] = turn(pack_f16(s[u][t][0], s[u][t][1]));
                    pb[u][t][1] = turn(pack_f16(s[u][t][2], s[u][t][3]));
                }

            // O^T: a lane's scales are those of tokens 2c, 2c + 1 and 2c + 8, 2c + 9.
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int v = 0; v < D / 16 / B::W; ++v) {
                    uint32_t vw[B::W];
                    shared_words<B::W>(at + u * S::BLOCK + B::VALUES + B::value_word(v * B::W, lane), vw);
#pragma unroll
                    for (int j = 0; j < B::W; j += 2) {
                        uint32_t vs[2]; // one group of 32 columns
                        shared_words<2>(at + u * S::BLOCK + B::VALUE_SCALES + 2 * B::value_scale(2 * c, (v * B::W + j) / 2), vs);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            uint32_t x[4];
                            f16x8(vw[j + e], x);
                            const uint32_t a[4] = {hmul2(x[0], vs[0]), hmul2(x[1], vs[0]), hmul2(x[2], vs[1]), hmul2(x[3], vs[1])};
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                mma16816(o[t][v * B::W + j + e], a, pb[u][t][0], pb[u][t][1]);
                        }
                    }
                }
            }
        };

        int i0 = seg.j0 + warp * step;
        if (pairs == 0 && next)
            begin(*next, stage_at);
        for (int k = 0; k < pairs; ++k, i0 += W * step) {
            __syncwarp(); // every lane is done with the last pair, whose place is the next copy's
            const bool more = k + 1 < pairs;
            if (more)
                copy(seg, k + 1, stage_at ^ 1, whole1);
            else if (next)
                begin(*next, stage_at ^ 1);
            const uint32_t at = ring + stage_at * S::STAGE;
            if (!mbar_wait(full + stage_at, parity, p.err, kErrWaitK)) {
                // Gives up (the host learns of it), but not before its copies under way are over,
                // or had their time.
                for (int wait = 0; wait < 2; ++wait) {
                    const uint64_t start = globaltimer_ns();
                    while (!mbar_try_wait(smem_u32(full + stage_at), parity) && globaltimer_ns() - start < kWaitLimitNs) {
                    }
                    if (!more)
                        break; // what the next segment has under way is waited for there
                    next_stage();
                }
                if (!more)
                    next_stage();
                else if (next)
                    begin(*next, stage_at);
                break;
            }
            next_stage();
            if (i0 < whole0 || i0 >= whole1)
                attend_pair(std::true_type(), at, i0);
            else
                attend_pair(std::false_type(), at, i0);
        }
        __syncwarp();
        const uint32_t groups = lost && lane < ROWS ? parts.lost[warp][lane] : 0u;
        __syncwarp(); // their place is the sums'

#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 4);
                sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 8);
                sum[t][h] += __shfl_xor_sync(0xffffffffu, sum[t][h], 16);
                const int r = 8 * t + 2 * c + h;
                if (g == 0) {
                    parts.m[warp][r] = none[t][h] ? -INFINITY : ref[t][h];
                    parts.l[warp][r] = sum[t][h];
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    parts.o[warp][r][16 * x + g] = o[t][x][h];
                    parts.o[warp][r][16 * x + 8 + g] = o[t][x][2 + h];
                }
            }
        if (lost) {
            __syncwarp();
            for (int r = 0; r < ROWS; ++r)
                for (uint32_t those = __shfl_sync(0xffffffffu, groups, r); those; those &= those - 1)
                    parts.o[warp][r][(__ffs(those) - 1) * kCacheGroup + lane] = NAN;
        }
    }

    // The warps' parts as one, m, l and four columns at a time of sum_i 2^(m_i - m) o_i, to
    // take(row, column, m, l, values).  All threads are past a barrier when this begins.
    template <typename F> __device__ __forceinline__ static void join(const Parts<D, NT> &parts, F &&take) {
        for (int x = threadIdx.x * 4; x < ROWS * D; x += W * 32 * 4) {
            const int r = x / D, col = x - r * D;
            float weight[W], mx = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w)
                mx = fmaxf(mx, weight[w] = parts.m[w][r]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = ex2_approx(weight[w] - base);
                const float4 o4 = *reinterpret_cast<const float4 *>(&parts.o[w][r][col]);
                l += f * parts.l[w][r];
                v.x += f * o4.x;
                v.y += f * o4.y;
                v.z += f * o4.z;
                v.w += f * o4.w;
            }
            take(r, col, mx, l, v);
        }
    }
};

// Barriers of the stages: each waits for the two lanes that copy a pair's blocks.
template <int N> __device__ __forceinline__ void make_bars(uint64_t *bars) {
    if (threadIdx.x < N)
        mbar_init(bars + threadIdx.x, 2);
    fence_mbarrier_init();
    fence_proxy_async_smem();
    __syncthreads();
}

// A cluster for each tile.
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(TokensShape<D, NT>::WARPS * 32, TokensShape<D, NT>::CTAS)
    window_e2m1_cluster_kernel(const __grid_constant__ TokensParams p) {
    using S = TokensShape<D, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[S::WARPS * S::STAGES];
    Parts<D, NT> &mine = *reinterpret_cast<Parts<D, NT> *>(smem + S::RING);
    const int parts = p.parts, pair = blockIdx.x / parts, part = blockIdx.x - pair * parts;
    Segment seg;
    seg.b = pair / p.kv_heads;
    seg.kvh = pair - seg.b * p.kv_heads;
    int n, m;
    lengths_of(p, seg.b, n, m);
    seg.tile = tile_of<S::ROWS>(p, n, m, blockIdx.y);
    seg.j0 = 2 * part;
    seg.j1 = seg.tile.blocks;
    make_bars<S::WARPS * S::STAGES>(bars);
    Worker<D, NT, BF16> worker(p, 2 * parts, smem, bars);
    worker.ask(seg);
    worker.load_queries(seg);
    worker.begin(seg, 0);
    worker.attend(seg, nullptr, mine);
    __syncthreads();
    worker.join(mine, [&](int r, int col, float m, float l, const float4 &v) {
        if (col == 0) {
            mine.cta_m[r] = m;
            mine.cta_l[r] = l;
        }
        *reinterpret_cast<float4 *>(&mine.o[0][r][col]) = v;
    });
    if (parts == 1) {
        __syncthreads();
        for (int x = threadIdx.x; x < S::ROWS * D; x += S::WARPS * 32) {
            const int r = x / D, col = x - r * D;
            if (r < seg.tile.rows && col < p.hd)
                store_out(p, seg.tile, seg.b, seg.kvh, r, col, mine.o[0][r][col], mine.cta_l[r]);
        }
        return;
    }
    // The CTAs' parts: their weights once for each row (over the ring, which is read), then each
    // CTA its share of the columns.
    float(*weight)[S::ROWS] = reinterpret_cast<float(*)[S::ROWS]>(smem), (*sums)[S::ROWS] = weight + kMaxParts;
    cluster_sync();
    for (int x = threadIdx.x; x < parts * S::ROWS; x += S::WARPS * 32) {
        const int k = x / S::ROWS, r = x - k * S::ROWS;
        weight[k][r] = peer_load(peer(&mine.cta_m[r], k));
        sums[k][r] = peer_load(peer(&mine.cta_l[r], k));
    }
    __syncthreads();
    if (threadIdx.x < S::ROWS) {
        const int r = threadIdx.x;
        float mx = -INFINITY, l = 0.f;
        for (int k = 0; k < parts; ++k)
            mx = fmaxf(mx, weight[k][r]);
        const float base = mx == -INFINITY ? 0.f : mx;
        for (int k = 0; k < parts; ++k) {
            const float f = ex2_approx(weight[k][r] - base);
            weight[k][r] = f;
            l += f * sums[k][r];
        }
        sums[0][r] = l;
    }
    __syncthreads();
    for (int x = part * S::WARPS * 32 + threadIdx.x; x < S::ROWS * D; x += parts * S::WARPS * 32) {
        const int r = x / D, col = x - r * D;
        if (r >= seg.tile.rows || col >= p.hd)
            continue;
        float v = 0.f;
#pragma unroll 4
        for (int k = 0; k < parts; ++k)
            v += weight[k][r] * peer_load(peer(&mine.o[0][r][col], k));
        store_out(p, seg.tile, seg.b, seg.kvh, r, col, v, sums[0][r]);
    }
    cluster_sync(); // no CTA leaves while another reads its part
}

// Quotients that mostly need 32 bits only.
__device__ __forceinline__ int quotient(long long a, long long b) {
    return (a | b) >> 32 ? static_cast<int>(a / b) : static_cast<int>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}
// Blocks of a CTA where `ctas` share `total`.
__device__ __forceinline__ long long share_of(long long total, int ctas) {
    const long long up = total + ctas - 1;
    return up >> 32 ? up / ctas : static_cast<long long>(static_cast<uint32_t>(up) / static_cast<uint32_t>(ctas));
}

// A tile that begins in a CTA's share of the list and ends in another's: for each CTA, behind
// the parts' slots.  parts 0: there is none.
struct alignas(16) SharedTile {
    int b = 0, kvh = 0, tile = 0, slot = 0, parts = 0, n = 0, m = 0, unused = 0;
};
template <int D, int NT> __device__ __forceinline__ SharedTile *shared_tile(const TokensParams &p, int cta) {
    return reinterpret_cast<SharedTile *>(p.parts_at + 2ll * p.ctas * TokensShape<D, NT>::SLOT) + cta;
}

// The list: blocks of the tiles, sequence after sequence, key head after key head, tile after
// tile.  CTA i takes blocks [i per, (i + 1) per).  The next segment's first blocks are on their
// way before the last ones of a segment are read.
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(TokensShape<D, NT>::WARPS * 32, TokensShape<D, NT>::CTAS)
    window_e2m1_list_kernel(const __grid_constant__ TokensParams p) {
    using S = TokensShape<D, NT>;
    constexpr int THREADS = S::WARPS * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[S::WARPS * S::STAGES];
    __shared__ long long place[S::WARPS];
    __shared__ Segment segments[32];
    __shared__ struct {
        long long at, tile; // where the next tile begins in the list, and its number
        int count;          // of the segments
    } walk;
    Parts<D, NT> &parts = *reinterpret_cast<Parts<D, NT> *>(smem + S::RING);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    make_bars<S::WARPS * S::STAGES>(bars);
    // Each thread has a run of sequences; the thread in whose run this CTA's first block is finds
    // the sequence and key head.
    const int run = (p.batch + THREADS - 1) / THREADS, b0 = threadIdx.x * run, b1 = min(p.batch, b0 + run);
    long long mine = 0;
    for (int b = b0; b < b1; ++b)
        mine += listed_of<S::ROWS>(p, b);
    mine *= p.kv_heads;
    long long before = mine;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, before, x);
        before += lane >= x ? y : 0;
    }
    if (lane == 31)
        place[warp] = before;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < S::WARPS; ++w) {
        before += w < warp ? place[w] : 0;
        total += place[w];
    }
    before -= mine;
    const long long per = share_of(total, gridDim.x);
    const long long from = blockIdx.x * per, to = min(total, from + per);
    if (threadIdx.x == 0)
        *shared_tile<D, NT>(p, blockIdx.x) = SharedTile{};
    if (from >= to)
        return;
    if (from >= before && from < before + mine) {
        int b = b0;
        long long of_head = listed_of<S::ROWS>(p, b);
        for (; b < b1 - 1 && from >= before + of_head * p.kv_heads; of_head = listed_of<S::ROWS>(p, b))
            before += of_head * p.kv_heads, ++b;
        // (Lengths that change under the kernel are a caller's mistake, but lead out of no array.)
        const int kvh = max(0, min(quotient(from - before, max(of_head, 1ll)), p.kv_heads - 1));
        walk.tile = (static_cast<long long>(b) * p.kv_heads + kvh) * p.tiles;
        walk.at = before + kvh * of_head;
    }
    // A warp works out 32 tiles at once, those of them that this CTA has a share in.
    const int of_sequence = p.kv_heads * p.tiles;
    auto refill = [&] {
        const long long at = walk.at, number = walk.tile + lane;
        const int b = quotient(number, of_sequence), in_b = static_cast<int>(number - static_cast<long long>(b) * of_sequence);
        Segment s;
        s.b = b;
        s.kvh = in_b / p.tiles;
        int size = 0, n, m;
        if (b < p.batch) {
            lengths_of(p, b, n, m);
            s.tile = tile_of<S::ROWS>(p, n, m, in_b - s.kvh * p.tiles);
            size = listed(s.tile);
        }
        uint32_t sum = size; // 32 tiles of at most 2^26 blocks
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, sum, x);
            sum += lane >= x ? y : 0;
        }
        const long long begin = at + (sum - size);
        const bool has = size && begin + size > from && begin < to;
        const uint32_t those = __ballot_sync(0xffffffffu, has);
        if (has) {
            const int j0 = static_cast<int>(max(from - begin, 0ll)), j1 = static_cast<int>(min(to - begin, static_cast<long long>(size)));
            s.j0 = max(j0 - kTileCost, 0);
            s.j1 = j1 - kTileCost;
            s.slot = j0 == 0 && j1 == size ? -1 : 2 * static_cast<int>(blockIdx.x) + (begin > from);
            segments[__popc(those & ((1u << lane) - 1))] = s;
            if (j0 == 0 && j1 < size) { // begins here, ends elsewhere: what the join needs to know
                SharedTile t;
                t.b = b;
                t.kvh = s.kvh;
                t.tile = in_b - s.kvh * p.tiles;
                t.slot = s.slot;
                t.n = s.tile.n;
                t.m = s.tile.m;
                t.parts = quotient(begin + size - 1, per) - static_cast<int>(blockIdx.x) + 1;
                *shared_tile<D, NT>(p, blockIdx.x) = t;
            }
        }
        __syncwarp();
        if (lane == 31) {
            walk.at = at + sum;
            walk.tile = number + 1;
            walk.count = __popc(those);
        }
    };
    Worker<D, NT, BF16> worker(p, 2, smem, bars);
    do {
        __syncthreads(); // walk and the segments are as they were left
        if (warp == 0)
            refill();
        __syncthreads();
        const int count = walk.count;
        if (count) {
            worker.ask(segments[0]);
            worker.load_queries(segments[0]);
            worker.begin(segments[0], worker.stage_at);
        }
        for (int i = 0; i < count; ++i) {
            const Segment &seg = segments[i], *next = i + 1 < count ? &segments[i + 1] : nullptr;
            worker.attend(seg, next, parts);
            if (next)
                worker.load_queries(*next);
            __syncthreads();
            if (seg.slot < 0) {
                worker.join(parts, [&](int r, int col, float, float l, const float4 &v) {
                    const float *e = &v.x;
                    if (r < seg.tile.rows)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (col + x < p.hd)
                                store_out(p, seg.tile, seg.b, seg.kvh, r, col + x, e[x], l);
                });
            } else {
                float *slot = p.parts_at + static_cast<long long>(seg.slot) * S::SLOT;
                worker.join(parts, [&](int r, int col, float m, float l, const float4 &v) {
                    if (col == 0)
                        *reinterpret_cast<float2 *>(slot + 2 * r) = make_float2(m, l);
                    *reinterpret_cast<float4 *>(slot + 2 * S::ROWS + r * D + col) = v;
                });
            }
            __syncthreads(); // the parts' place is free
        }
    } while (walk.at < to && walk.tile < static_cast<long long>(p.batch) * of_sequence);
}

// Joins the parts of the tiles that several CTAs share: a CTA for each of the list's, and two
// rows of the tile that begins there (few tiles of many parts would meet in few SMs otherwise:
// 131072 keys x 8 heads, 75 parts each, 40 us so and 59 with eight rows, 64 x up to 16384 keys
// 122 either way).  A part's weight is worked out once for a row; SHARES threads share a
// column's parts.
constexpr int kJoinThreads = 256, kJoinParts = 1024, kJoinRows = 2;
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) window_e2m1_join_kernel(const __grid_constant__ TokensParams p) {
    using S = TokensShape<D, NT>;
    constexpr int FOURS = kJoinRows * D / 4, SHARES = kJoinThreads / FOURS;
    __shared__ float weight[kJoinRows][kJoinParts], sums[kJoinRows][kJoinParts], total_l[kJoinRows];
    __shared__ __align__(16) float share[SHARES - 1][kJoinRows * D];
    asm volatile("griddepcontrol.wait;" ::: "memory"); // every CTA: this grid's end stands for the list's as well
    const SharedTile what = *shared_tile<D, NT>(p, blockIdx.x);
    const int parts = what.parts, row0 = blockIdx.y * kJoinRows;
    if (parts == 0)
        return;
    const Tile tile = tile_of<S::ROWS>(p, what.n, what.m, what.tile);
    const int rows = min(kJoinRows, tile.rows - row0), b = what.b, kvh = what.kvh;
    if (rows <= 0)
        return;
    // Its first part is where the tile began, the others are first parts of their CTAs.
    const float *from = p.parts_at + static_cast<long long>(what.slot) * S::SLOT;
    const float *others = p.parts_at + 2ll * blockIdx.x * S::SLOT;
    auto slot = [&](int c) { return c ? others + 2ll * c * S::SLOT : from; };
    // The first parts' columns are on their way while the weights are worked out.
    constexpr int EARLY = 6;
    const int of = threadIdx.x / FOURS, x = threadIdx.x % FOURS * 4, r = x / D, col = x % D;
    const bool mine = of < SHARES && r < rows;
    auto columns = [&](int c) { return *reinterpret_cast<const float4 *>(slot(c) + 2 * S::ROWS + row0 * D + x); };
    float4 early[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
        if (mine && of + i * SHARES < parts)
            early[i] = columns(of + i * SHARES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < rows) {
        float mx = -INFINITY, l = 0.f;
        for (int c = lane; c < parts; c += 32) {
            const float2 ml = *reinterpret_cast<const float2 *>(slot(c) + 2 * (row0 + warp));
            weight[warp][c] = ml.x;
            sums[warp][c] = ml.y;
            mx = fmaxf(mx, ml.x);
        }
#pragma unroll
        for (int x = 16; x; x >>= 1)
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        const float base = mx == -INFINITY ? 0.f : mx;
        for (int c = lane; c < parts; c += 32) {
            const float f = ex2_approx(weight[warp][c] - base);
            weight[warp][c] = f;
            l += f * sums[warp][c];
        }
#pragma unroll
        for (int x = 16; x; x >>= 1)
            l += __shfl_xor_sync(0xffffffffu, l, x);
        if (lane == 0)
            total_l[warp] = l;
    }
    __syncthreads();
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
        auto add = [&](const float4 &o, float f) {
            v[0] += f * o.x;
            v[1] += f * o.y;
            v[2] += f * o.z;
            v[3] += f * o.w;
        };
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            if (of + i * SHARES < parts)
                add(early[i], weight[r][of + i * SHARES]);
#pragma unroll 4
        for (int c = of + EARLY * SHARES; c < parts; c += SHARES)
            add(columns(c), weight[r][c]);
        if (of)
            *reinterpret_cast<float4 *>(&share[of - 1][x]) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    if (of || !mine)
        return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int k = 0; k < SHARES - 1; ++k)
            v[e] += share[k][x + e];
        if (col + e < p.hd)
            store_out(p, tile, b, kvh, row0 + r, col + e, v[e], total_l[r]);
    }
}

template <int D, int NT, bool BF16> int launch_rows(const TokensParams &p, cudaStream_t stream) {
    using S = TokensShape<D, NT>;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.blockDim = dim3(S::WARPS * 32);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (p.parts) {
        static std::atomic<unsigned long long> done{0};
        const void *kernel = reinterpret_cast<const void *>(window_e2m1_cluster_kernel<D, NT, BF16>);
        cudaError_t e = set_smem_limit(kernel, S::SMEM, done);
        if (e == cudaSuccess && p.parts > 8) // clusters above 8 CTAs need the kernel's consent
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess)
            return static_cast<int>(e);
        cfg.gridDim = dim3(static_cast<unsigned>(p.parts) * p.batch * p.kv_heads, p.tiles);
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = p.parts;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        return static_cast<int>(cudaLaunchKernelEx(&cfg, window_e2m1_cluster_kernel<D, NT, BF16>, p));
    }
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = set_smem_limit(reinterpret_cast<const void *>(window_e2m1_list_kernel<D, NT, BF16>), S::SMEM, done);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    cfg.gridDim = dim3(p.ctas);
    cfg.numAttrs = 0;
    e = cudaLaunchKernelEx(&cfg, window_e2m1_list_kernel<D, NT, BF16>, p);
    if (e != cudaSuccess)
        return static_cast<int>(e);
    // The join is set up while the list's kernel runs, and waits for its end before it reads the parts.
    cfg.gridDim = dim3(p.ctas, S::ROWS / kJoinRows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, window_e2m1_join_kernel<D, NT>, p));
}
template <int D> int launch_d(const TokensParams &p, int rows, bool bf16, cudaStream_t stream) {
    if (rows == 8)
        return bf16 ? launch_rows<D, 1, true>(p, stream) : launch_rows<D, 1, false>(p, stream);
    if (rows == 16)
        return bf16 ? launch_rows<D, 2, true>(p, stream) : launch_rows<D, 2, false>(p, stream);
    return bf16 ? launch_rows<D, 3, true>(p, stream) : launch_rows<D, 3, false>(p, stream);
}

// How a call is split: rows of a tile, CTAs of a cluster, or (parts 0) of the list.
struct Split {
    int rows, tiles, parts, ctas;
    size_t workspace;
    double us; // about what it takes
};
Split split_in(const WindowE2m1Args &a, int rows_of_tile) {
    const CacheArgs &c = a.cache;
    const long long rows = static_cast<long long>(a.heads / c.kv_heads) * c.q_len;
    Split s;
    s.rows = rows_of_tile;
    s.tiles = static_cast<int>((rows + s.rows - 1) / s.rows);
    long long keys = a.kv_len;
    if (a.window > 0)
        keys = std::min(keys, static_cast<long long>(a.window) + c.q_len + a.right + a.sinks);
    const long long of_tile = (keys + kCacheBlock - 1) / kCacheBlock + 1;
    const long long tiles = static_cast<long long>(s.tiles) * c.batch * c.kv_heads;
    const long long most = std::min<long long>(kJoinParts, 1ll * ctas_of_sm(cache_width(c.hd), s.rows) * fmha_sm_count()); // CTAs at once
    s.parts = 1;
    // (Clusters of 16 with 24 rows do not all fit at once: 2 x 2048 keys, 20 rows, 23 us with 16, 12 with 8.)
    const int most_parts = s.rows == 24 ? 8 : kMaxParts;
    while (s.parts < most_parts && tiles * s.parts * 2 <= most && of_tile >= 2ll * s.parts * 8)
        s.parts *= 2;
    // In microseconds, as measured: a CTA's blocks one after another, slower the more rows they
    // meet and the more CTAs share its SM; the list has its second kernel on top, but also evens
    // out sequences that are shorter than kv_len, which is not known here, and gets a tenth for
    // that (clusters of several rounds even them out themselves).  Measured, cluster / list, 8 key heads of 128, one row of four heads: 1 x 8192 keys
    // 10.5 / 13.5, 1 x 32768 22.7 / 19.9, 1 x 65536 39.6 / 25.7, 16 x 4096 15.9 / 22.1, 64 x 2048
    // 26.0 / 32.0, 64 x up to 4096 46.9 / 45.3, 64 x up to 16384 165 / 123.  Narrow heads with many
    // rows are underrated: 8 x 128 queries over 128 keys, 16 heads of 64, take 18.9 us here and 13.6
    // by the prompts' kernel, heads of 32 15.6 and 12.3 (heads of 128 15.2 either way).
    const double sms = fmha_sm_count(), ctas = static_cast<double>(tiles) * s.parts;
    const double block = (s.rows == 8 ? 1.0 : s.rows == 16 ? 1.3 : 1.7) * (0.1 + 0.9 * cache_width(c.hd) / 128);
    const double rounds = std::max(1.0, ctas / most);
    const double cluster = 1 + 4 * rounds + block * of_tile / s.parts * rounds * (0.11 + 0.028 * std::min(ctas, static_cast<double>(most)) / sms);
    const double total = static_cast<double>(tiles) * (of_tile + kTileCost);
    s.ctas = static_cast<int>(std::min<double>(most, std::ceil(total / 32)));
    const double list = 13 + block * total / s.ctas * (0.11 + 0.028 * s.ctas / sms);
    s.workspace = 0;
    s.us = std::min(list, cluster);
    if (list < (rounds < 2 ? 1.1 : 1.0) * cluster) {
        s.parts = 0;
        s.workspace = s.ctas * (2ull * s.rows * (cache_width(c.hd) + 2) * 4 + sizeof(SharedTile));
    }
    return s;
}
// The cheapest height of a tile: high ones convert a block for more rows, low ones have more CTAs
// and warps.  Measured, 8 / 16 / 24 rows: 1 x 8192 keys, 16 rows 11.8 / 13.3 us, 64 rows 20.1 /
// 20.4 / 23.0; 2 x 2048, 20 rows 8.8 / 11.5 / 12.6; 16 x 4096 of 8192, 20 rows 47 / 52 / 40; 1 x
// 131072, 16 rows 62 / 51.
Split split_of(const WindowE2m1Args &a) {
    const long long rows = static_cast<long long>(a.heads / a.cache.kv_heads) * a.cache.q_len;
    Split best = split_in(a, 8);
    for (int height = 16; height <= 24 && rows > height - 8; height += 8) {
        const Split s = split_in(a, height);
        if (s.us < best.us)
            best = s;
    }
    return best;
}

} // namespace

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
    p.group_inv = ((1u << 20) + p.group - 1) / p.group;
    p.q_len = c.q_len;
    p.kv_len = a.kv_len;
    p.hd = c.hd;
    p.window = a.window;
    p.right = a.right;
    p.sinks = a.sinks;
    p.out_dtype = a.out_dtype;
    const double scale = a.scale > 0 ? a.scale : 1.0 / std::sqrt(static_cast<double>(c.hd));
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    const Split split = split_of(a);
    p.parts = split.parts;
    p.ctas = split.ctas;
    p.tiles = split.tiles;
    p.batch = c.batch;
    p.parts_at = static_cast<float *>(a.workspace);
    p.err = a.err;
    const bool bf16 = a.dtype == kBF16;
    switch (cache_width(c.hd)) {
    case 32:
        return launch_d<32>(p, split.rows, bf16, stream);
    case 64:
        return launch_d<64>(p, split.rows, bf16, stream);
    case 96:
        return launch_d<96>(p, split.rows, bf16, stream);
    default:
        return launch_d<128>(p, split.rows, bf16, stream);
    }
}

// Few rows read the cache as it is; for others the keys and values go back to 16 bits in the
// workspace (exactly), and the prompts' kernel reads them.  What each takes, in microseconds as
// measured: the prompts' kernel has blocks of 128 rows, whose steps of 64 keys come one after
// another, in rounds of what the SMs hold.  Measured, few rows / prompts, 32/8 heads of 128: one
// sequence of 8192 keys, 16 queries 23 / 109; 32
// queries 36 / 109, 128 queries 81 / 109; 16 of up to 4096 keys, 32 queries 103 / 128, 64 queries
// 155 / 129; one of 1024 keys, 100 queries 20 / 22.
static bool few_rows(const WindowE2m1Args &a) {
    const CacheArgs &c = a.cache;
    if (static_cast<long long>(a.heads / c.kv_heads) * c.q_len > kMostRows)
        return false;
    double keys = a.kv_len;
    if (a.window > 0)
        keys = std::min<double>(keys, static_cast<double>(a.window) + c.q_len + a.right + a.sinks);
    const double steps = std::min<double>(a.kv_len, keys + 127) / 64 + 1;
    const double blocks = static_cast<double>(c.batch) * a.heads * ((c.q_len + 127) / 128);
    const double read = 2.0 * c.batch * c.kv_heads * keys * c.hd * 2.6 / 4e6;
    const double prompt = 10 + read + 0.7 * steps * std::max(1.0, blocks / (1.45 * fmha_sm_count()));
    return split_of(a).us <= prompt;
}

size_t window_e2m1_workspace(const WindowE2m1Args &a) {
    if (few_rows(a))
        return split_of(a).workspace;
    return 4ull * a.cache.batch * a.cache.kv_heads * a.kv_len * a.cache.hd;
}

int window_e2m1_launch(const WindowE2m1Args &a, cudaStream_t stream) {
    if (few_rows(a))
        return window_e2m1_tokens_launch(a, stream);
    const size_t bytes = window_e2m1_workspace(a);
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
    w.lift = a.dtype == kF16 ? kTop : 0.f;
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
