// Matrix product of rows with rows, out = act(scale_a * scale_w * (a w^T) + bias) + residual: the entry
// point and the kernel for operands of any alignment.
//
// k_linear_any: tiles of 64 x 64 results per CTA, 4 x 4 per thread, operands staged through shared memory
// 32 columns at a time with one load per element.  int8 sums are exact in int32, 16-bit ones accumulate in
// float32 in the order of k.  Bound: the FMA pipes and its scalar loads; it exists for rows that do not
// start on 16-byte boundaries, which the tensor-core kernels' copies cannot read.
#include "linear.cuh"

namespace lk {

constexpr int AT = 64, AK = 32;

template <typename T>
struct AnyAcc {
    using type = float;
    static __device__ __forceinline__ float wide(T v) { return Elem<T>::get(v); }
};
template <>
struct AnyAcc<signed char> {
    using type = int;
    static __device__ __forceinline__ int wide(signed char v) { return v; }
};

template <typename T>
__global__ void __launch_bounds__(256) k_linear_any(const LinearArgs p, long long tiles_n) {
    using Acc = typename AnyAcc<T>::type;
    __shared__ Acc sa[AK][AT + 1], sw[AK][AT + 1];
    const long long i0 = (blockIdx.x / tiles_n) * AT, j0 = (blockIdx.x % tiles_n) * AT;
    const int ti = (threadIdx.x / 16) * 4, tj = (threadIdx.x % 16) * 4;
    const T *a = static_cast<const T *>(p.a), *w = static_cast<const T *>(p.w);
    Acc acc[4][4] = {};
    for (long long k0 = 0; k0 < p.k; k0 += AK) {
#pragma unroll
        for (int s = 0; s < AT * AK / 256; ++s) {
            const int e = s * 256 + (int)threadIdx.x, r = e / AK, c = e % AK;
            const bool in = k0 + c < p.k;
            sa[c][r] = in && i0 + r < p.m ? AnyAcc<T>::wide(a[(i0 + r) * p.lda + k0 + c]) : Acc(0);
            sw[c][r] = in && j0 + r < p.n ? AnyAcc<T>::wide(w[(j0 + r) * p.ldw + k0 + c]) : Acc(0);
        }
        __syncthreads();
#pragma unroll 8
        for (int c = 0; c < AK; ++c) {
            Acc x[4], y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = sa[c][ti + u], y[u] = sw[c][tj + u];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[u][v] += x[u] * y[v];
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (i0 + ti + u < p.m && j0 + tj + v < p.n) finish_one(p, i0 + ti + u, j0 + tj + v, (float)acc[u][v]);
}

template <typename T>
static int any_launch(const LinearArgs &p, cudaStream_t st) {
    const long long tm = (p.m + AT - 1) / AT, tn = (p.n + AT - 1) / AT;
    if (tm > 0x7fffffffll / tn) return fail(LK_ERANGE, "lk_linear: more result tiles than a grid holds");
    return launch("lk_linear", k_linear_any<T>, (unsigned)(tm * tn), 256, st, p, tn);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_linear(int device, int dtype, int64_t m, int64_t n, int64_t k, const void *d_a, int64_t lda,
                         const float *d_a_scales, const void *d_w, int64_t ldw, const float *d_w_scales,
                         const void *d_bias, int act, const void *d_residual, int64_t ldr,
                         int out_dtype, void *d_out, int64_t ldo, void *stream) {
    if (dtype != LK_I8 && dtype != LK_F16 && dtype != LK_BF16)
        return fail(LK_EINVAL, "lk_linear: dtype is LK_I8, LK_F16 or LK_BF16");
    if (!float_type(out_dtype)) return fail(LK_EINVAL, "lk_linear: out_dtype is LK_F32, LK_F16 or LK_BF16");
    if (act < LK_ACT_NONE || act > LK_ACT_GELU_TANH) return fail(LK_EINVAL, "lk_linear: unknown activation");
    if (m < 0 || n < 0 || k < 0) return fail(LK_EINVAL, "lk_linear: bad size");
    if (k > LK_LINEAR_MAX_K) return fail(LK_ERANGE, "lk_linear: k is limited to LK_LINEAR_MAX_K (65536)");
    if (m > 0x7fffffff || n > 0x7fffffff) return fail(LK_ERANGE, "lk_linear: more than 2^31-1 rows");
    const bool some = m > 0 && n > 0;
    if (some && (!d_out || (k > 0 && (!d_a || !d_w)))) return fail(LK_EINVAL, "lk_linear: NULL pointer");
    if ((m > 1 && ((k > 0 && lda < k) || ldo < n || (d_residual && ldr < n))) || (n > 1 && k > 0 && ldw < k))
        return fail(LK_EINVAL, "lk_linear: a row stride is smaller than the row");
    const int eb = type_bytes(dtype), ob = type_bytes(out_dtype);
    const auto off = [](const void *p, int to) { return reinterpret_cast<uintptr_t>(p) % to != 0; };
    if (off(d_a, eb) || off(d_w, eb) || off(d_a_scales, 4) || off(d_w_scales, 4) || off(d_bias, ob) || off(d_residual, ob) || off(d_out, ob))
        return fail(LK_EINVAL, "lk_linear: a pointer is not aligned to its element type");
    DeviceScope scope;
    LK_TRY(scope.enter(device, "lk_linear"));
    if (!some) return LK_OK;
    const LinearArgs p = {d_a, d_w, d_a_scales, d_w_scales, d_bias, d_residual, d_out, m, n, k, lda, ldw, ldr, ldo, act, out_dtype};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (linear_mma_reads(p, dtype)) return linear_mma_launch(p, dtype, device, st);
    if (dtype == LK_I8) return any_launch<signed char>(p, st);
    if (dtype == LK_F16) return any_launch<__half>(p, st);
    return any_launch<__nv_bfloat16>(p, st);
}

extern "C" int lk_ops_status(int device) {
    DeviceScope scope;
    LK_TRY(scope.enter(device, "lk_ops_status"));
    LK_CUDA(cudaDeviceSynchronize());  // streams that the legacy default stream does not wait for, too
    int linear = 0, norm = 0;
    LK_TRY(linear_failed(&linear));
    LK_TRY(norm_failed(&norm));
    if (linear) return fail(LK_ETIMEOUT, "lk_linear: a bounded wait inside the kernel ran out; its results are not complete");
    if (norm) return fail(LK_ETIMEOUT, "lk_rms_norm_i8: a bounded wait inside the kernel ran out; its results are not complete");
    return LK_OK;
}
