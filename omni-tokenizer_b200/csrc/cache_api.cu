// cache_api.cu -- extern "C" entry points of the rotary positions, the 4-bit key/value
// cache and the attention over it, declared in include/omni_b200.h.
#include "omni_b200.h"

#include "cache_e2m1.cuh"
#include "fmha.h"
#include "layer.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cuda_runtime.h>

namespace omni_b200 {
// ops_api.cu
int ctx_fail(int code, const char *msg);
void ctx_clear();
int *kernel_error_word();
int launch_status(int rc, const char *what);

namespace {
constexpr int kMost = 1 << 30;
constexpr long long kMostStride = 1ll << 38;

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t type_bytes(int dtype) { return dtype == OMNI_B200_F32 ? 4 : 2; }

// Strides (batch, head, token) of a tensor [batch, heads, tokens, width]; that of a single
// element is never used.  False: one is out of range, or no multiple of `unit`.
bool take_strides(const int64_t *strides, int batch, int heads, int tokens, int width, int unit, long long (&to)[3]) {
    const int sizes[3] = {batch, heads, tokens};
    const long long row = std::max(1, tokens) * static_cast<long long>(width), plain[3] = {std::max(1, heads) * row, row, width};
    for (int d = 0; d < 3; ++d) {
        to[d] = strides && sizes[d] > 1 ? strides[d] : (plain[d] + unit - 1) / unit * unit;
        if (to[d] < width || (sizes[d] > 1 && to[d] > kMostStride) || to[d] % unit)
            return false;
    }
    return true;
}

// The cache's own arguments; NULL, or what is wrong with them.
const char *take_cache(const omni_b200_cache_e2m1 *c, const int32_t *lengths, const int32_t *q_lengths, int batch,
                       int kv_heads, int q_len, int head_dim, CacheArgs &a) {
    if (!c)
        return "null cache";
    if (batch < 0 || q_len < 0 || kv_heads <= 0 || q_len > kMost)
        return "sizes must be positive and at most 2^30";
    if (head_dim <= 0 || head_dim > 128 || head_dim % 8)
        return "head_dim must be a multiple of 8 in [8, 128]";
    if (c->pages <= 0 || c->page_tokens <= 0 || c->page_tokens % kCacheBlock || c->page_tokens > kMost)
        return "a cache needs pages of a multiple of 16 tokens, at most 2^30";
    const int width = c->table ? c->table_width : 1;
    if (width <= 0 || static_cast<long long>(width) * c->page_tokens > kMost)
        return "a sequence's pages must hold 1 to 2^30 tokens";
    if (!c->table && c->pages < batch)
        return "without a table the cache needs a page for each sequence";
    const long long bytes = static_cast<long long>(c->page_tokens / kCacheBlock) * static_cast<long long>(cache_block_bytes(head_dim));
    const long long head = kv_heads > 1 ? c->head_stride : bytes, page = c->pages > 1 ? c->page_stride : bytes * kv_heads;
    if (head < bytes || page < bytes || head > kMostStride || page > kMostStride || head % 16 || page % 16)
        return "page and head strides must be multiples of 16 bytes, at least a page of a head and at most 2^38";
    a.data = c->data;
    a.table = c->table;
    a.pages = c->pages;
    a.page_tokens = c->page_tokens;
    a.table_width = width;
    a.page_stride = page;
    a.head_stride = head;
    a.lengths = lengths;
    a.q_lengths = q_lengths;
    a.batch = batch;
    a.kv_heads = kv_heads;
    a.q_len = q_len;
    a.hd = head_dim;
    return nullptr;
}
// What is wrong with its pointers, where there is work.
const char *bad_pointers(const CacheArgs &a) {
    if (!a.data || !a.lengths)
        return "null pointer";
    if (!aligned(a.data, 16) || !aligned(a.table, 4) || !aligned(a.lengths, 4) || !aligned(a.q_lengths, 4))
        return "the cache must be 16-byte aligned, its table and the lengths to their type";
    return nullptr;
}
int refuse(const char *what, const char *why, int code = 1) {
    static thread_local char text[200];
    std::snprintf(text, sizeof(text), "%s: %s", what, why);
    return ctx_fail(code, text);
}

int cache_rows(const char *what, bool read, const void *k, const void *v, const omni_b200_cache_e2m1 *cache,
               const int32_t *lengths, const int32_t *q_lengths, int batch, int kv_heads, int q_len, int head_dim,
               const int64_t *strides, int dtype, void *stream) {
    ctx_clear();
    if (dtype != OMNI_B200_BF16 && dtype != OMNI_B200_F16 && !(read && dtype == OMNI_B200_F32))
        return refuse(what, read ? "dtype must be F32, BF16 or F16" : "dtype must be BF16 or F16");
    CacheArgs a;
    if (const char *why = take_cache(cache, lengths, q_lengths, batch, kv_heads, q_len, head_dim, a))
        return refuse(what, why);
    if (static_cast<double>(batch) * kv_heads * ((q_len + 30.) / 16) > 4.0 * kMost)
        return refuse(what, "more than 2^32 blocks of 16 tokens", 4);
    long long ks[3], vs[3];
    const int unit = 16 / static_cast<int>(type_bytes(dtype));
    if (!take_strides(strides, batch, kv_heads, q_len, head_dim, unit, ks) ||
        !take_strides(strides ? strides + 3 : nullptr, batch, kv_heads, q_len, head_dim, unit, vs))
        return refuse(what, "strides must be at least head_dim, at most 2^38, and multiples of 16 bytes");
    if (batch == 0 || q_len == 0)
        return 0;
    if (!k || !v)
        return refuse(what, "null pointer");
    if (const char *why = bad_pointers(a))
        return refuse(what, why);
    if (!aligned(k, 16) || !aligned(v, 16))
        return refuse(what, "k and v must be 16-byte aligned");
    if (!kernel_error_word())
        return refuse(what, "no CUDA device", 7);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch_status(read ? cache_read_launch(a, const_cast<void *>(k), const_cast<void *>(v), ks, vs, dtype, CacheReadRange(), s)
                              : cache_write_launch(a, k, v, ks, vs, dtype, s),
                         what);
}
} // namespace
} // namespace omni_b200

using namespace omni_b200;

extern "C" {

int omni_b200_rotary(const void *q, void *q_out, const void *k, void *k_out, const void *positions,
                     const void *frequencies, const uint8_t *axes, int batch, int heads, int kv_heads, int tokens,
                     int head_dim, int pairs, int n_axes, const int64_t *strides, const int64_t *position_strides,
                     int adjacent, int inverse, int position_type, int frequency_f64, int dtype, void *stream) {
    ctx_clear();
    if (dtype < OMNI_B200_F32 || dtype > OMNI_B200_F16)
        return ctx_fail(1, "rotary: dtype must be F32, BF16 or F16");
    if (position_type < kPositionI32 || position_type > kPositionF32)
        return ctx_fail(1, "rotary: position_type must be I32, I64 or F32");
    if (batch < 0 || tokens < 0 || heads <= 0 || heads > 65535 || kv_heads < 0 || kv_heads > 65535 || head_dim <= 0)
        return ctx_fail(1, "rotary: sizes must be positive, heads and kv_heads at most 65535");
    if (pairs <= 0 || pairs > kMaxPairs || 2 * pairs > head_dim || head_dim > 65536)
        return ctx_fail(1, "rotary: pairs must be in [1, 256] and 2 * pairs at most head_dim, which is at most 65536");
    if (n_axes <= 0 || n_axes > 256)
        return ctx_fail(1, "rotary: n_axes must be in [1, 256]");
    for (int i = 0; axes && i < pairs; ++i)
        if (axes[i] >= n_axes)
            return ctx_fail(1, "rotary: an axis of axes is not below n_axes");
    if (static_cast<double>(batch) * tokens * head_dim > 256.0 * kMost)
        return ctx_fail(4, "rotary: more than 2^38 columns of tokens");
    const bool has_k = k || k_out;
    RotaryArgs a;
    if (!take_strides(strides, batch, heads, tokens, head_dim, 1, a.qs) ||
        !take_strides(strides ? strides + 3 : nullptr, batch, heads, tokens, head_dim, 1, a.qos) ||
        (has_k && (!take_strides(strides ? strides + 6 : nullptr, batch, kv_heads, tokens, head_dim, 1, a.ks) ||
                   !take_strides(strides ? strides + 9 : nullptr, batch, kv_heads, tokens, head_dim, 1, a.kos))))
        return ctx_fail(1, "rotary: strides must be at least head_dim and at most 2^38");
    for (int d = 0; d < 3; ++d) {
        a.ps[d] = position_strides ? position_strides[d] : d == 0 ? static_cast<long long>(batch) * tokens : d == 1 ? tokens : 1;
        if (a.ps[d] < 0 || a.ps[d] > kMostStride)
            return ctx_fail(1, "rotary: position strides must be in [0, 2^38]");
    }
    if (batch == 0 || tokens == 0)
        return 0;
    if (!q || !q_out || !positions || !frequencies || (has_k && (!k || !k_out || kv_heads == 0)))
        return ctx_fail(1, "rotary: null pointer, or k without key heads");
    const size_t size = type_bytes(dtype);
    if (!aligned(q, size) || !aligned(q_out, size) || !aligned(k, size) || !aligned(k_out, size) ||
        !aligned(positions, position_type == kPositionI64 ? 8 : 4) ||
        !aligned(frequencies, frequency_f64 ? 8 : 4))
        return ctx_fail(1, "rotary: a pointer is not aligned to its element type");
    if (q_out == k_out || q_out == k || (has_k && k_out == q))
        return ctx_fail(1, "rotary: q_out and k_out must be apart, and each overlap no input but its own");
    if ((q == q_out && !std::equal(a.qs, a.qs + 3, a.qos)) || (has_k && k == k_out && !std::equal(a.ks, a.ks + 3, a.kos)))
        return ctx_fail(1, "rotary: an output in its input's place must have its strides");
    a.q = q;
    a.k = k;
    a.q_out = q_out;
    a.k_out = k_out;
    a.positions = positions;
    a.frequencies = frequencies;
    a.axes = axes;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.tokens = tokens;
    a.hd = head_dim;
    a.pairs = pairs;
    a.position_type = position_type;
    a.dtype = dtype;
    a.frequency_f64 = frequency_f64 != 0;
    a.adjacent = adjacent != 0;
    a.inverse = inverse != 0;
    if (!kernel_error_word())
        return ctx_fail(7, "rotary: no CUDA device");
    return launch_status(rotary_launch(a, static_cast<cudaStream_t>(stream)), "rotary");
}

size_t omni_b200_cache_e2m1_bytes(size_t tokens, int head_dim) {
    if (head_dim <= 0 || head_dim > 128 || head_dim % 8 || tokens == 0 || tokens % kCacheBlock || tokens > kMost)
        return 0;
    return tokens / kCacheBlock * cache_block_bytes(head_dim);
}

int omni_b200_cache_write_e2m1(const void *k, const void *v, const omni_b200_cache_e2m1 *cache, const int32_t *lengths,
                               const int32_t *q_lengths, int batch, int kv_heads, int q_len, int head_dim,
                               const int64_t *strides, int dtype, void *stream) {
    return cache_rows("cache_write_e2m1", false, k, v, cache, lengths, q_lengths, batch, kv_heads, q_len, head_dim,
                      strides, dtype, stream);
}

int omni_b200_cache_read_e2m1(const omni_b200_cache_e2m1 *cache, void *k, void *v, const int32_t *lengths,
                              const int32_t *q_lengths, int batch, int kv_heads, int q_len, int head_dim,
                              const int64_t *strides, int dtype, void *stream) {
    return cache_rows("cache_read_e2m1", true, k, v, cache, lengths, q_lengths, batch, kv_heads, q_len, head_dim,
                      strides, dtype, stream);
}

// Sizes that both the query of the workspace and the call check; NULL where they are right.
static const char *window_sizes(int heads, int kv_heads, int q_len, int window, int right, int sinks, int batch) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads)
        return "heads must be a multiple of kv_heads";
    if (window > kMost || right < 0 || right > kMost || sinks < 0 || sinks > kMost)
        return "window, right and sinks must be at most 2^30, right and sinks not negative";
    if (static_cast<double>(batch) * heads * ((q_len + 127) / 128) > kMost)
        return "more than 2^30 blocks of queries";
    return nullptr;
}

size_t omni_b200_attention_window_e2m1_workspace(int batch, int heads, int kv_heads, int q_len, int kv_len,
                                                 int head_dim, int window, int right, int sinks) {
    if (batch <= 0 || q_len <= 0 || q_len > kMost || kv_len <= 0 || kv_len > kMost || head_dim <= 0 || head_dim > 128 ||
        head_dim % 8 || window_sizes(heads, kv_heads, q_len, window, right, sinks, batch))
        return 0;
    WindowE2m1Args a;
    a.cache.batch = batch;
    a.cache.kv_heads = kv_heads;
    a.cache.q_len = q_len;
    a.cache.hd = head_dim;
    a.heads = heads;
    a.kv_len = kv_len;
    a.window = window;
    a.right = std::min(right, kMost - 1);
    a.sinks = sinks;
    return window_e2m1_workspace(a);
}

int omni_b200_attention_window_e2m1(const void *q, const omni_b200_cache_e2m1 *cache, void *out,
                                    const int32_t *lengths, const int32_t *q_lengths, int batch, int heads,
                                    int kv_heads, int q_len, int kv_len, int head_dim, const int64_t *strides,
                                    int window, int right, int sinks, float scale, int dtype, int out_dtype,
                                    void *workspace, size_t workspace_bytes, void *stream) {
    constexpr const char *what = "attention_window_e2m1";
    ctx_clear();
    if (dtype != OMNI_B200_BF16 && dtype != OMNI_B200_F16)
        return refuse(what, "dtype must be BF16 or F16");
    if (out_dtype != dtype && out_dtype != OMNI_B200_F32)
        return refuse(what, "out_dtype must be dtype or F32");
    WindowE2m1Args a;
    if (const char *why = take_cache(cache, lengths, q_lengths, batch, kv_heads, q_len, head_dim, a.cache))
        return refuse(what, why);
    if (const char *why = window_sizes(heads, kv_heads, q_len, window, right, sinks, batch))
        return refuse(what, why);
    if (kv_len <= 0 || kv_len > a.cache.capacity())
        return refuse(what, "kv_len must be positive and at most what a sequence's pages hold");
    if (std::isnan(scale) || std::isinf(scale))
        return refuse(what, "scale must be finite");
    if (!take_strides(strides, batch, heads, q_len, head_dim, 8, a.qs) ||
        !take_strides(strides ? strides + 3 : nullptr, batch, heads, q_len, head_dim, 1, a.os))
        return refuse(what, "strides must be at least head_dim, at most 2^38, and those of q multiples of 8");
    if (batch == 0 || q_len == 0)
        return 0;
    if (!q || !out)
        return refuse(what, "null pointer");
    if (const char *why = bad_pointers(a.cache))
        return refuse(what, why);
    if (!aligned(q, 16) || !aligned(out, type_bytes(out_dtype)))
        return refuse(what, "q must be 16-byte aligned, out to its element type");
    a.q = q;
    a.out = out;
    a.heads = heads;
    a.kv_len = kv_len;
    a.window = window;
    a.right = std::min(right, kMost - 1); // as good as kMost, and a position + right + 1 fits in 32 bits
    a.sinks = sinks;
    a.dtype = dtype;
    a.out_dtype = out_dtype;
    a.scale = scale;
    a.workspace = workspace;
    const size_t need = window_e2m1_workspace(a);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return refuse(what, "the workspace is too small, or not 16-byte aligned");
    a.err = kernel_error_word();
    if (!a.err)
        return refuse(what, "no CUDA device", 7);
    return launch_status(window_e2m1_launch(a, static_cast<cudaStream_t>(stream)), what);
}

} // extern "C"
