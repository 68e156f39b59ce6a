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

__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
        case LK_ACT_RELU: return v < 0.0f ? 0.0f : v;  // NaN stays
        case LK_ACT_SILU: return v / (1.0f + __expf(-v));
        case LK_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        case LK_ACT_GELU_TANH: {
            // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
            const float z = 0.79788456080286536f * (v + 0.044715f * v * v * v);
            return v / (1.0f + __expf(-2.0f * z));
        }
        default: return v;
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
    v = activate(p.act, v);
    if (p.residual != nullptr) v += load_as(p.out_type, p.residual, i * p.ldr + j);
    store_as(p.out_type, p.out, i * p.ldo + j, v);
}

}  // namespace lk
