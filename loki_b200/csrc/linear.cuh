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

// The activation of N values: one branch for all of them.
template <int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
    if (act == LK_ACT_RELU) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = v[u] < 0.0f ? 0.0f : v[u];  // NaN stays
    } else if (act == LK_ACT_SILU) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = __fdividef(v[u], 1.0f + __expf(-v[u]));
    } else if (act == LK_ACT_GELU) {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = 0.5f * v[u] * (1.0f + erff(v[u] * 0.70710678118654752f));
    } else if (act == LK_ACT_GELU_TANH) {
        // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float z = 0.79788456080286536f * (v[u] + 0.044715f * v[u] * v[u] * v[u]);
            v[u] = __fdividef(v[u], 1.0f + __expf(-2.0f * z));
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
    activate_all<1>(p.act, y);
    if (p.residual != nullptr) y[0] += load_as(p.out_type, p.residual, i * p.ldr + j);
    store_as(p.out_type, p.out, i * p.ldo + j, y[0]);
}

// linear_mma.cu: whether the tensor-core kernel's copies can read these operands, and its launch.
bool linear_mma_reads(const LinearArgs &p, int dtype);
int linear_mma_launch(const LinearArgs &p, int dtype, int device, cudaStream_t st);
// Whether one of its bounded waits ran out on the current device since the last call; waits for the device.
int linear_failed(int *out);

}  // namespace lk
