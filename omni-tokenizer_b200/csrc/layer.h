// layer.h -- host-side interfaces of the 8-bit layer kernels (rms_norm.cu,
// linear_e4m3_sm100.cu).  Each launch returns 0, a CUDA error code, -1 (no
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

} // namespace omni_b200
