// layer.h -- host-side interfaces of the layer kernels (rms_norm.cu, linear_e4m3_sm100.cu,
// rotary.cu, cache_e2m1.cu, window_e2m1_tokens.cu).  Each launch returns 0, a CUDA error code, -1 (no
// tensor-map entry point) or 1000 + CUresult.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace omni_b200 {

// SMs of the device (fmha_sm100.cu; looked up once).
int fmha_sm_count();

// Element types of the layer operators (the values of omni_b200_dtype).
enum : int { kF32 = 0, kBF16 = 1, kF16 = 2, kE4M3 = 3 };

struct RowsArgs {
    const void *x = nullptr, *residual = nullptr, *weight = nullptr;
    void *residual_out = nullptr, *out = nullptr;
    float *scales = nullptr; // e4m3 output: [rows, ceil(cols / 128)]
    long long rows = 0;
    int cols = 0;
    long long x_stride = 0, residual_stride = 0, residual_out_stride = 0, out_stride = 0; // elements
    float eps = 0.f;
    int dtype = kBF16;
    bool norm = false;      // false: quantise x as it is
    bool quantize = false;  // e4m3 output with scales, else dtype
    int *err = nullptr;     // the device's error word
};
int rows_launch(const RowsArgs &a, cudaStream_t stream);

// 128 x 128 blocks of [rows, cols]: e4m3 q and scales [ceil(rows/128), ceil(cols/128)].
int quantize_blocks_launch(const void *x, void *q, float *scales, long long rows, int cols,
                           long long x_stride, long long q_stride, int dtype, cudaStream_t stream);

struct LinearArgs {
    const void *a = nullptr, *w = nullptr; // e4m3 [m, k], [n, k]
    const float *a_scales = nullptr, *w_scales = nullptr;
    const void *bias = nullptr; // [n] of out_dtype
    void *out = nullptr;        // [m, n]
    int m = 0, n = 0, k = 0;
    long long lda = 0, ldw = 0, ldo = 0;
    int out_dtype = kBF16;
    int *err = nullptr;
};
int linear_e4m3_launch(const LinearArgs &a, cudaStream_t stream);

// Types of rotary positions (the values of omni_b200_position_type).
enum : int { kPositionI32 = 0, kPositionI64 = 1, kPositionF32 = 2 };
constexpr int kMaxPairs = 256;

// omni_b200_rotary: strides in elements (batch, head, token), of positions (axis, batch, token).
struct RotaryArgs {
    const void *q = nullptr, *k = nullptr; // k may be absent
    void *q_out = nullptr, *k_out = nullptr;
    long long qs[3] = {}, ks[3] = {}, qos[3] = {}, kos[3] = {}, ps[3] = {};
    const void *positions = nullptr, *frequencies = nullptr;
    const uint8_t *axes = nullptr; // host, [pairs]
    int batch = 0, heads = 0, kv_heads = 0, tokens = 0, hd = 0, pairs = 0;
    int position_type = kPositionI32, dtype = kBF16;
    bool frequency_f64 = false, adjacent = false, inverse = false;
};
int rotary_launch(const RotaryArgs &a, cudaStream_t stream);

// A 4-bit key/value cache (cache_e2m1.cuh) and its operators' arguments.
struct CacheArgs {
    void *data = nullptr;
    const int *table = nullptr;
    const int *lengths = nullptr, *q_lengths = nullptr;
    int pages = 0, page_tokens = 0, table_width = 0; // table_width 1 where there is no table
    long long page_stride = 0, head_stride = 0;      // bytes
    int batch = 0, kv_heads = 0, q_len = 0, hd = 0;
    long long capacity() const { return static_cast<long long>(page_tokens) * table_width; }
};
// k and v [batch, kv_heads, q_len, hd], strides (batch, head, token) in elements.
int cache_write_launch(const CacheArgs &c, const void *k, const void *v, const long long (&ks)[3],
                       const long long (&vs)[3], int dtype, cudaStream_t stream);
// A sequence's last rows, from row 0 of k and v on; or (prompt) all its rows that a query of
// attention_window sees, each at its own place.
struct CacheReadRange {
    bool whole = false;
    int kv_len = 0, window = 0, sinks = 0;
};
int cache_read_launch(const CacheArgs &c, void *k, void *v, const long long (&ks)[3], const long long (&vs)[3],
                      int dtype, const CacheReadRange &range, cudaStream_t stream);

// omni_b200_attention_window_e2m1.
struct WindowE2m1Args {
    CacheArgs cache;
    const void *q = nullptr;
    void *out = nullptr;
    long long qs[3] = {}, os[3] = {};
    int heads = 0, kv_len = 0;
    int window = 0, right = 0, sinks = 0;
    int dtype = kBF16, out_dtype = kBF16;
    float scale = 0.f; // 0: hd^-1/2
    void *workspace = nullptr;
    int *err = nullptr;
};
// Bytes of workspace (16-byte aligned) for these sizes, 0: none is used.
size_t window_e2m1_workspace(const WindowE2m1Args &a);
int window_e2m1_launch(const WindowE2m1Args &a, cudaStream_t stream);
// Its kernel for few rows (window_e2m1_tokens.cu).
int window_e2m1_tokens_launch(const WindowE2m1Args &a, cudaStream_t stream);

} // namespace omni_b200
