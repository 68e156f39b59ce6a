// Matrix product of rows with rows and its epilogue: arguments and the arithmetic behind the sum, shared
// by the kernels of linear.cu and linear_mma.cu.
#pragma once
#include "devops.cuh"

namespace lk {

struct LinearArgs {
    const void *a, *w;
    const float *a_scales, *w_scales;  // NULL = ones
    const void *bias, *residual;       // out_type, NULL = none
    void *out;
    long long m, n, k, lda, ldw, ldr, ldo;
    int act, out_type;
};

// The share of a normal distribution beyond a, 0 <= a <= 20: exp(-a^2 / 2) P(t), t = 1 / (1 + 0.295 a), with P fitted (weighted least
// squares after Lawson) to exp(a^2 / 2) erfc(a / sqrt 2) / 2, 4e-8 relative.  1 + erf, which is twice this, cancels below 0.
// FULL: within 14 * 2^-24 relative, with t corrected (to 2^-24; P is 2.7 times as sensitive to it) and what a^2 lost brought back in.
// Else those two are left out, 2^-24 * (27 + 4 a^2 / 2).  With erfcf in its place 4,096 x 8,192 x 1,024 bf16 took 130 us instead of 90.
template <bool FULL>
__device__ __forceinline__ float normal_tail(float a) {
    const float d = fmaf(0.295f, a, 1.0f), h = a * a;
    float t = __fdividef(1.0f, d);
    if (FULL) t = fmaf(t, fmaf(-fmaf(0.295f, a, 1.0f - d), t, fmaf(-d, t, 1.0f)), t);
    float p = 0.0392500758f;
    p = fmaf(p, t, -0.182633162f), p = fmaf(p, t, 0.269538283f), p = fmaf(p, t, -0.11551214f), p = fmaf(p, t, 0.165299833f);
    p = fmaf(p, t, 0.0851306245f), p = fmaf(p, t, 0.121609196f), p = fmaf(p, t, 0.117300875f), p = fmaf(p, t, 1.6388547e-05f);
    if (FULL) return p * expf(-0.5f * h) * fmaf(-0.5f, fmaf(a, a, -h), 1.0f);  // the last: what h lost
    return p * __expf(-0.5f * h);
}

// v / (1 + exp(-t)), t of v's sign.  FULL: to 12 * 2^-24, also where the exponential of -t would pass float32's range (v < -88 of SiLU); else
// with the fast exponential and quotient, 2^-24 * 8 (1 + |t|).
template <bool FULL>
__device__ __forceinline__ float gated(float v, float t) {
    if (!FULL) return __fdividef(v, 1.0f + __expf(-t));
    const float e = expf(-fabsf(t));
    return __fdividef(t < 0.0f ? v * e : v, 1.0f + e);  // 2 ulp; a division rounded to half of one took 20 % longer over a small product
}

// The activation of N values: one branch for all of them.  FULL for float32 results; 16-bit ones hold fewer bits than what is saved.
template <bool FULL, int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
    if (act == LK_ACT_RELU) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = v[u] < 0.0f ? 0.0f : v[u];  // NaN stays
    } else if (act == LK_ACT_SILU) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = gated<FULL>(v[u], v[u]);
    } else if (act == LK_ACT_GELU) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float q = normal_tail<FULL>(fminf(fabsf(v[u]), 20.0f));
            v[u] *= v[u] < 0.0f ? q : 1.0f - q;
        }
    } else if (act == LK_ACT_GELU_TANH) {
        // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float z = 0.79788456080286536f * (v[u] + 0.044715f * v[u] * v[u] * v[u]);
            v[u] = gated<FULL>(v[u], 2.0f * z);
        }
    }
}

__device__ __forceinline__ float scale_of(const float *s, long long i) { return s != nullptr ? s[i] : 1.0f; }

__device__ __forceinline__ void store_as(int dtype, void *p, long long i, float v) {
    if (dtype == LK_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == LK_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// One value of the result from its finished sum.
__device__ __forceinline__ void finish_one(const LinearArgs &p, long long i, long long j, float acc) {
    float v = acc * (scale_of(p.a_scales, i) * scale_of(p.w_scales, j));
    if (p.bias != nullptr) v += load_as(p.out_type, p.bias, j);
    float y[1] = {v};
    if (p.out_type == LK_F32) activate_all<true>(p.act, y);
    else activate_all<false>(p.act, y);
    if (p.residual != nullptr) y[0] += load_as(p.out_type, p.residual, i * p.ldr + j);
    store_as(p.out_type, p.out, i * p.ldo + j, y[0]);
}

// linear_mma.cu: whether the tensor-core kernel's copies can read these operands, and its launch.
bool linear_mma_reads(const LinearArgs &p, int dtype);
int linear_mma_launch(const LinearArgs &p, int dtype, int device, cudaStream_t st);
// Whether one of its bounded waits ran out on the current device since the last call; waits for the device.
int linear_failed(int *out);

}  // namespace lk
