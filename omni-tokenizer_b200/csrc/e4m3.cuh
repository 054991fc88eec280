// e4m3.cuh -- element conversions shared by the 8-bit layer kernels.
//
// Quantisation of a group with largest magnitude amax:
//   scale = max(amax / 448, 2^-126),  q = e4m3(x / scale),
// so x ~ q * scale.  448 is e4m3's largest value.  The floor 2^-126 keeps
// 1 / scale finite for a group of zeros (whose q are zeros).  A NaN does not
// take part in amax and becomes e4m3's NaN; an infinity makes the scale
// infinite, and the group then stands for NaN.
// Inputs of 16 bits often have quotients half way between two e4m3 values, so what
// is quantised as it is (EXACT) takes x * (1 / scale) with one correction by its
// residual (Markstein, 1990), which rounds as a division would, for two more
// operations on a pair of elements (24000 x 4304: 53 -> 56 us; 24000 x 4096: 49
// either way).  A norm's values carry fp32
// rounding errors of their own and do without: of 27 million 17 round otherwise than in
// 64 bits, 19 with fp32 divisions, and the correction costs 16384 x 8192 148 -> 165 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100.cuh"

namespace omni_b200 {

constexpr int kGroup = 128; // columns (of weights: columns and rows) that share a scale
constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f; // 2^-126

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements as they lie in memory (16 bytes of a 2-byte type,
// 32 of fp32), and as fp32.
template <typename T> struct Vec8 {
    uint4 w[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Vec8<T> load8(const T *p) {
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        v.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return v;
}
template <typename T> __device__ __forceinline__ void store8(T *p, const Vec8<T> &v) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        reinterpret_cast<uint4 *>(p)[i] = v.w[i];
}
template <typename T> __device__ __forceinline__ void unpack8(const Vec8<T> &v, float (&f)[8]) {
    const T *e = reinterpret_cast<const T *>(v.w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        f[i] = to_float(e[i]);
}
template <typename T> __device__ __forceinline__ Vec8<T> pack8(const float (&f)[8]) {
    Vec8<T> v;
    T *e = reinterpret_cast<T *>(v.w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        e[i] = from_float<T>(f[i]);
    return v;
}

// Two e4m3 values in 16 bits, `lo` in the low byte (round to nearest even,
// beyond 448 to 448, NaN to NaN).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// A group's divisor.
struct Divisor {
    float scale, inv; // scale 0 stands for an infinite one: no correction
    template <bool EXACT> __device__ __forceinline__ float quotient(float x) const {
        const float q = x * inv;
        return EXACT ? fmaf(fmaf(-q, scale, x), inv, q) : q;
    }
};
__device__ __forceinline__ Divisor divisor_of(float scale) {
    Divisor d;
    d.scale = scale <= 3.402823466e38f ? scale : 0.f;
    d.inv = __frcp_rn(scale);
    return d;
}
template <bool EXACT> __device__ __forceinline__ uint2 e4m3x8(const float (&f)[8], const Divisor &d) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) { // two elements an instruction
        if constexpr (EXACT) {
            float e0, e1;
            fmul2(q[i], q[i + 1], f[i], f[i + 1], d.inv, d.inv);
            ffma2(e0, e1, q[i], q[i + 1], -d.scale, -d.scale, f[i], f[i + 1]);
            ffma2(q[i], q[i + 1], e0, e1, d.inv, d.inv, q[i], q[i + 1]);
        } else {
            fmul2(q[i], q[i + 1], f[i], f[i + 1], d.inv, d.inv);
        }
    }
    uint2 r;
    r.x = e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16);
    r.y = e4m3x2(q[4], q[5]) | (e4m3x2(q[6], q[7]) << 16);
    return r;
}
__device__ __forceinline__ float amax8(const float (&f)[8]) {
    const float a = fmax3(fabsf(f[0]), fabsf(f[1]), fabsf(f[2])), b = fmax3(fabsf(f[3]), fabsf(f[4]), fabsf(f[5]));
    return fmaxf(fmax3(a, b, fabsf(f[6])), fabsf(f[7]));
}
__device__ __forceinline__ float group_scale(float amax) {
    return fmaxf(__fdiv_rn(amax, kE4m3Max), kMinScale);
}

} // namespace omni_b200
