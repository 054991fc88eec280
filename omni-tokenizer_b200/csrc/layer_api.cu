// layer_api.cu -- extern "C" entry points of the 8-bit layer operators and the
// windowed attention declared in include/omni_b200.h.
#include "omni_b200.h"

#include "fmha.h"
#include "layer.h"

#include <algorithm>
#include <cmath>
#include <cuda_runtime.h>

namespace omni_b200 {
// ops_api.cu
int ctx_fail(int code, const char *msg);
void ctx_clear();
int *kernel_error_word();
int launch_status(int rc, const char *what);

namespace {
bool element_type(int dtype) { return dtype >= OMNI_B200_F32 && dtype <= OMNI_B200_F16; }
bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
size_t type_bytes(int dtype) { return dtype == OMNI_B200_F32 ? 4 : 2; }
constexpr size_t kMaxRows = 1ull << 40, kMaxCols = 1ull << 24, kMaxStride = 1ull << 40;
} // namespace
} // namespace omni_b200

using namespace omni_b200;

extern "C" {

int omni_b200_rms_norm(const void *x, const void *residual, const void *weight, void *residual_out, void *out,
                       float *scales, size_t rows, size_t cols, size_t x_stride, size_t residual_stride,
                       size_t residual_out_stride, size_t out_stride, float eps, int dtype, int out_dtype,
                       void *stream) {
    ctx_clear();
    if (!element_type(dtype))
        return ctx_fail(1, "rms_norm: dtype must be F32, BF16 or F16");
    if (out_dtype != dtype && out_dtype != OMNI_B200_E4M3)
        return ctx_fail(1, "rms_norm: out_dtype must be dtype or E4M3");
    const bool quantize = out_dtype == OMNI_B200_E4M3;
    if (quantize != (scales != nullptr) && rows)
        return ctx_fail(1, "rms_norm: scales belong to an E4M3 output, and it needs them");
    if (rows && (!x || !weight || !out))
        return ctx_fail(1, "rms_norm: null pointer");
    if (rows && (residual == nullptr) != (residual_out == nullptr))
        return ctx_fail(1, "rms_norm: residual and residual_out go together");
    if (cols == 0 || cols > kMaxCols || rows > kMaxRows)
        return ctx_fail(1, "rms_norm: cols must be in [1, 2^24]");
    if (!(eps >= 0.f) || std::isinf(eps))
        return ctx_fail(1, "rms_norm: eps must be finite and not negative");
    if (x_stride < cols || out_stride < cols || x_stride > kMaxStride || out_stride > kMaxStride ||
        (residual && (residual_stride < cols || residual_out_stride < cols || residual_stride > kMaxStride ||
                      residual_out_stride > kMaxStride)))
        return ctx_fail(1, "rms_norm: a row stride is smaller than cols, or above 2^40");
    if (rows && (out == residual_out || (quantize && (out == x || out == residual))))
        return ctx_fail(1, "rms_norm: out must not be residual_out, nor, in E4M3, an input");
    if (rows > 1 && ((residual && ((residual_out == x && residual_out_stride != x_stride) ||
                                   (residual_out == residual && residual_out_stride != residual_stride) ||
                                   (out == residual && out_stride != residual_stride))) ||
                     (out == x && out_stride != x_stride)))
        return ctx_fail(1, "rms_norm: an output in an input's place must have its row stride");
    const size_t size = type_bytes(dtype);
    if (!aligned(x, size) || !aligned(residual, size) || !aligned(weight, size) || !aligned(residual_out, size) ||
        !aligned(out, quantize ? 1 : size) || !aligned(scales, 4))
        return ctx_fail(1, "rms_norm: a pointer is not aligned to its element type");
    if (rows == 0)
        return 0;
    RowsArgs a;
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.residual_out = residual_out;
    a.out = out;
    a.scales = scales;
    a.rows = static_cast<long long>(rows);
    a.cols = static_cast<int>(cols);
    a.x_stride = static_cast<long long>(x_stride);
    a.residual_stride = static_cast<long long>(residual_stride);
    a.residual_out_stride = static_cast<long long>(residual_out_stride);
    a.out_stride = static_cast<long long>(out_stride);
    a.eps = eps;
    a.dtype = dtype;
    a.norm = true;
    a.quantize = quantize;
    a.err = kernel_error_word();
    if (!a.err)
        return ctx_fail(7, "rms_norm: no CUDA device");
    return launch_status(rows_launch(a, static_cast<cudaStream_t>(stream)), "rms_norm");
}

int omni_b200_quantize_e4m3(const void *x, void *q, float *scales, size_t rows, size_t cols, size_t x_stride,
                            size_t q_stride, int block_rows, int dtype, void *stream) {
    ctx_clear();
    if (!element_type(dtype))
        return ctx_fail(1, "quantize_e4m3: dtype must be F32, BF16 or F16");
    if (block_rows != 1 && block_rows != 128)
        return ctx_fail(1, "quantize_e4m3: block_rows must be 1 or 128");
    if (rows && (!x || !q || !scales))
        return ctx_fail(1, "quantize_e4m3: null pointer");
    if (cols == 0 || cols > kMaxCols || rows > (block_rows == 1 ? kMaxRows : 65535u * 128u))
        return ctx_fail(1, "quantize_e4m3: cols must be in [1, 2^24], rows of 128-row blocks at most 8388480");
    if (x_stride < cols || q_stride < cols || x_stride > kMaxStride || q_stride > kMaxStride)
        return ctx_fail(1, "quantize_e4m3: a row stride is smaller than cols, or above 2^40");
    if (!aligned(x, type_bytes(dtype)) || !aligned(scales, 4))
        return ctx_fail(1, "quantize_e4m3: a pointer is not aligned to its element type");
    if (rows == 0)
        return 0;
    if (block_rows == 128)
        return launch_status(quantize_blocks_launch(x, q, scales, static_cast<long long>(rows), static_cast<int>(cols),
                                                    static_cast<long long>(x_stride), static_cast<long long>(q_stride),
                                                    dtype, static_cast<cudaStream_t>(stream)),
                             "quantize_e4m3");
    RowsArgs a;
    a.x = x;
    a.out = q;
    a.scales = scales;
    a.rows = static_cast<long long>(rows);
    a.cols = static_cast<int>(cols);
    a.x_stride = static_cast<long long>(x_stride);
    a.out_stride = static_cast<long long>(q_stride);
    a.dtype = dtype;
    a.quantize = true;
    a.err = kernel_error_word();
    if (!a.err)
        return ctx_fail(7, "quantize_e4m3: no CUDA device");
    return launch_status(rows_launch(a, static_cast<cudaStream_t>(stream)), "quantize_e4m3");
}

int omni_b200_linear_e4m3(const void *a, const float *a_scales, const void *w, const float *w_scales,
                          const void *bias, void *out, size_t m, size_t n, size_t k, size_t lda, size_t ldw,
                          size_t ldo, int out_dtype, void *stream) {
    ctx_clear();
    if (!element_type(out_dtype))
        return ctx_fail(1, "linear_e4m3: out_dtype must be F32, BF16 or F16");
    if (n == 0 || k == 0 || n > (1u << 22) || k > kMaxCols || m > (1u << 30))
        return ctx_fail(1, "linear_e4m3: n must be in [1, 2^22], k in [1, 2^24], m at most 2^30");
    if (m == 0)
        return 0;
    if (!a || !a_scales || !w || !w_scales || !out)
        return ctx_fail(1, "linear_e4m3: null pointer");
    if (lda < k || ldw < k || ldo < n || lda > kMaxStride / 2 || ldw > kMaxStride / 2 || ldo > kMaxStride / 8)
        return ctx_fail(1, "linear_e4m3: a row stride is smaller than its row, or above 2^37");
    if (lda % 16 || ldw % 16 || !aligned(a, 16) || !aligned(w, 16))
        return ctx_fail(1, "linear_e4m3: a and w must be 16-byte aligned, lda and ldw multiples of 16");
    const size_t size = type_bytes(out_dtype);
    if (!aligned(out, size) || !aligned(bias, size) || !aligned(a_scales, 4) || !aligned(w_scales, 4))
        return ctx_fail(1, "linear_e4m3: a pointer is not aligned to its element type");
    if (((m + 127) / 128) * ((n + 255) / 256) > (1u << 30))
        return ctx_fail(4, "linear_e4m3: out has more than 2^30 tiles");
    LinearArgs l;
    l.a = a;
    l.w = w;
    l.a_scales = a_scales;
    l.w_scales = w_scales;
    l.bias = bias;
    l.out = out;
    l.m = static_cast<int>(m);
    l.n = static_cast<int>(n);
    l.k = static_cast<int>(k);
    l.lda = static_cast<long long>(lda);
    l.ldw = static_cast<long long>(ldw);
    l.ldo = static_cast<long long>(ldo);
    l.out_dtype = out_dtype;
    l.err = kernel_error_word();
    if (!l.err)
        return ctx_fail(7, "linear_e4m3: no CUDA device");
    return launch_status(linear_e4m3_launch(l, static_cast<cudaStream_t>(stream)), "linear_e4m3");
}

int omni_b200_attention_window(const void *q, const void *k, const void *v, void *out, int batch, int heads,
                               int kv_heads, int q_len, int kv_len, int head_dim, const int64_t *strides,
                               const int32_t *lengths, const int32_t *q_lengths, int window, int right, int sinks,
                               float scale, int dtype, int out_dtype, void *stream) {
    ctx_clear();
    constexpr int kMost = 1 << 30;
    if (dtype != OMNI_B200_BF16 && dtype != OMNI_B200_F16)
        return ctx_fail(1, "attention_window: dtype must be BF16 or F16");
    if (out_dtype != dtype && out_dtype != OMNI_B200_F32)
        return ctx_fail(1, "attention_window: out_dtype must be dtype or F32");
    if (batch < 0 || q_len < 0 || heads <= 0 || kv_heads <= 0 || kv_len <= 0 || q_len > kMost || kv_len > kMost)
        return ctx_fail(1, "attention_window: sizes must be positive and at most 2^30");
    if (heads % kv_heads)
        return ctx_fail(1, "attention_window: heads must be a multiple of kv_heads");
    if (head_dim <= 0 || head_dim > 128 || head_dim % 8)
        return ctx_fail(4, "attention_window: head_dim must be a multiple of 8 in [8, 128]");
    if (window > kMost || right < 0 || right > kMost || sinks < 0 || sinks > kMost)
        return ctx_fail(1, "attention_window: window, right and sinks must be at most 2^30, right and sinks not negative");
    if (std::isnan(scale) || std::isinf(scale))
        return ctx_fail(1, "attention_window: scale must be finite");
    if (static_cast<double>(batch) * heads * ((q_len + 127) / 128) > kMost)
        return ctx_fail(4, "attention_window: more than 2^30 blocks of queries");
    if (batch == 0 || q_len == 0)
        return 0;
    if (!q || !k || !v || !out)
        return ctx_fail(1, "attention_window: null tensor pointer");
    WindowArgs a;
    const int of_heads[4] = {heads, kv_heads, kv_heads, heads}, of_len[4] = {q_len, kv_len, kv_len, q_len};
    long long *to[4] = {a.qs, a.ks, a.vs, a.os};
    for (int i = 0; i < 4; ++i) {
        const int sizes[3] = {batch, of_heads[i], of_len[i]};
        const long long plain[3] = {static_cast<long long>(of_heads[i]) * of_len[i] * head_dim,
                                    static_cast<long long>(of_len[i]) * head_dim, head_dim};
        for (int d = 0; d < 3; ++d) {
            // The stride of a single element is never used.
            to[i][d] = strides && sizes[d] > 1 ? strides[3 * i + d] : plain[d];
            if (to[i][d] < head_dim || to[i][d] > (1ll << 38) || (i < 3 && to[i][d] % 8))
                return ctx_fail(1, "attention_window: strides must be at least head_dim, at most 2^38, and those of "
                                   "q, k and v multiples of 8");
        }
    }
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16))
        return ctx_fail(1, "attention_window: q, k and v must be 16-byte aligned");
    if (!aligned(out, type_bytes(out_dtype)) || !aligned(lengths, 4) || !aligned(q_lengths, 4))
        return ctx_fail(1, "attention_window: a pointer is not aligned to its element type");
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.batch = batch;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.q_len = q_len;
    a.kv_len = kv_len;
    a.hd = head_dim;
    a.lengths = lengths;
    a.q_lengths = q_lengths;
    a.window = window;
    a.right = std::min(right, kMost - 1); // as good as kMost, and a position + right + 1 fits in 32 bits
    a.sinks = sinks;
    a.bf16 = dtype == OMNI_B200_BF16;
    a.out_dtype = out_dtype;
    a.scale = scale;
    a.err = kernel_error_word();
    if (!a.err)
        return ctx_fail(7, "attention_window: no CUDA device");
    return launch_status(attention_window(a, static_cast<cudaStream_t>(stream)), "attention_window");
}

} // extern "C"
