// Root-mean-square norm of x (+ residual) with an int8 output, one scale per row.
//
//   h = x + r;  y = h * inv * g with inv = 1 / sqrt(mean(h^2) + eps);  s = max|y| / 127;  c = round(y / s)
//
// inv is one positive number per row, so with p = h * g:  max|y| = inv * max|p| and y / s = 127 p / max|p|.
// The codes do not need inv at all, and both reductions of a row (the sum of h^2 and the maximum of
// |p|) are taken in ONE meeting of its threads, from values that stay in registers: x and r are read once,
// the sum and the codes written once.
//
// Bound: HBM (x, r and the sum at their types, one byte of code per element).
#include <cfloat>

#include "devops.cuh"

namespace lk {

struct NormArgs {
    const void *x, *r, *gain;
    void *sum;
    signed char *codes;
    float *scales;
    long long rows, ldx, ldr, lds, ldc;
    int dim, gain_type;
    float eps;
};

// Sum of squares in float64: float32 squares overflow from |h| = 1.8e19 on, and a row's sum is then
// exact to the last bits in any order.
struct RowStat {
    double ss;
    unsigned top;  // bits of max|p|: ordered like the values, NaN above infinity
};

__device__ __forceinline__ RowStat merge(RowStat a, RowStat b) { return {a.ss + b.ss, max(a.top, b.top)}; }

__device__ __forceinline__ RowStat warp_stat(RowStat s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.ss += __shfl_xor_sync(0xffffffffu, s.ss, o);
    s.top = __reduce_max_sync(0xffffffffu, s.top);
    return s;
}

constexpr unsigned kInfBits = 0x7f800000u;

// THREADS threads of a CTA share a row; a thread holds V groups of eight elements.  VEC: groups are eight
// consecutive elements read by 16-byte loads (rows on 16-byte boundaries); else element e of the row
// belongs to thread e % THREADS, one load each.
template <typename T, int THREADS, int V, bool VEC>
__global__ void __launch_bounds__(THREADS) k_rms_norm_i8(const NormArgs a) {
    __shared__ RowStat part[32];
    __shared__ double slow_top[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const T *r = static_cast<const T *>(a.r) + row * a.ldr;
    T *sum = static_cast<T *>(a.sum) + row * a.lds;
    signed char *codes = a.codes + row * a.ldc;
    const int dim = a.dim;

    // place of element i of this thread's group v
    auto at = [&](int v, int i) { return VEC ? (v * THREADS + tid) * 8 + i : (v * 8 + i) * THREADS + tid; };
    float h[V][8], p[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (VEC && at(v, 0) + 8 <= dim) {
            load8(x + at(v, 0), h[v]);
            if (a.r != nullptr) {
                float rv[8];
                load8(r + at(v, 0), rv);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[v][i] += rv[i];
            }
            if (a.sum != nullptr) store8(sum + at(v, 0), h[v]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = at(v, i);
                h[v][i] = 0.0f;
                if (e < dim) {
                    h[v][i] = Elem<T>::get(x[e]);
                    if (a.r != nullptr) h[v][i] += Elem<T>::get(r[e]);
                    if (a.sum != nullptr) sum[e] = Elem<T>::put(h[v][i]);
                }
            }
        }
    }
    RowStat st = {0.0, 0u};
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = at(v, i);
            const float g = (a.gain != nullptr && e < dim) ? load_as(a.gain_type, a.gain, e) : 1.0f;
            p[v][i] = h[v][i] * g;
            st.ss = fma((double)h[v][i], (double)h[v][i], st.ss);
            st.top = max(st.top, __float_as_uint(p[v][i]) & 0x7fffffffu);
        }
    }
    st = warp_stat(st);
    if (THREADS > 32) {
        if (lane == 0) part[warp] = st;
        __syncthreads();
        st = part[0];
#pragma unroll
        for (int w = 1; w < THREADS / 32; ++w) st = merge(st, part[w]);
    }
    const bool finite = st.ss < CUDART_INF;  // false for NaN too
    const double inv = rsqrt(st.ss / dim + (double)a.eps);
    float scale;
    if (finite && st.top != 0u && (st.top >= kInfBits || st.top < 0x0d800000u)) {
        // h * g leaves the comfortable range of float32 (overflow, or max|p| below 2^-100): the same in float64
        double top = 0.0;
        bool nan = false;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = at(v, i);
                const double q = (double)h[v][i] * ((a.gain != nullptr && e < dim) ? (double)load_as(a.gain_type, a.gain, e) : 1.0);
                top = fmax(top, fabs(q));
                nan |= !(fabs(q) < CUDART_INF);
            }
        if (nan) top = CUDART_INF;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (THREADS > 32) {
            if (lane == 0) slow_top[warp] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < THREADS / 32; ++w) top = fmax(top, slow_top[w]);
        }
        scale = (float)(top * inv / 127.0);
        const bool good = scale < CUDART_INF_F && top < CUDART_INF;
        if (!good) scale = CUDART_NAN_F;
        const double step = good ? 127.0 / top : 0.0;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = at(v, i);
                const double q = (double)h[v][i] * ((a.gain != nullptr && e < dim) ? (double)load_as(a.gain_type, a.gain, e) : 1.0);
                if (e < dim) codes[e] = good ? (signed char)(int)rint(fmin(fmax(q * step, -127.0), 127.0)) : (signed char)0;
            }
    } else {
        float step;
        if (!finite) {
            scale = CUDART_NAN_F;
            step = 0.0f;
        } else if (st.top == 0u) {  // nothing but zeros
            scale = step = 0.0f;
        } else {
            const float top = __uint_as_float(st.top);
            scale = (float)((double)top * inv) / 127.0f;
            step = 127.0f / top;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            alignas(8) signed char c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // a row without a step gets zeros whatever its values are (0 * NaN is not 0)
                const float q = step == 0.0f ? 0.0f : fminf(fmaxf(rintf(p[v][i] * step), -127.0f), 127.0f);
                c[i] = (signed char)(int)q;
            }
            if (VEC && at(v, 0) + 8 <= dim) {
                *reinterpret_cast<uint2 *>(codes + at(v, 0)) = *reinterpret_cast<const uint2 *>(c);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at(v, i) < dim) codes[at(v, i)] = c[i];
            }
        }
    }
    if (tid == 0) a.scales[row] = scale;
}

template <typename T, bool VEC>
static int norm_launch(const NormArgs &a, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    const int groups = (a.dim + 7) / 8;
    if (groups <= 32) return launch("lk_rms_norm_i8", k_rms_norm_i8<T, 32, 1, VEC>, grid, 32, st, a);
    if (groups <= 128) return launch("lk_rms_norm_i8", k_rms_norm_i8<T, 128, 1, VEC>, grid, 128, st, a);
    if (groups <= 512) return launch("lk_rms_norm_i8", k_rms_norm_i8<T, 256, 2, VEC>, grid, 256, st, a);
    if (groups <= 1024) return launch("lk_rms_norm_i8", k_rms_norm_i8<T, 512, 2, VEC>, grid, 512, st, a);
    return launch("lk_rms_norm_i8", k_rms_norm_i8<T, 1024, 4, VEC>, grid, 1024, st, a);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_rms_norm_i8(int device, int dtype, int64_t rows, int dim, const void *d_x, int64_t ldx,
                              const void *d_residual, int64_t ldr, const void *d_gain, int gain_dtype, float eps,
                              void *d_sum, int64_t lds, int8_t *d_codes, int64_t ldc, float *d_scales, void *stream) {
    if (!float_type(dtype) || (d_gain && !float_type(gain_dtype)))
        return fail(LK_EINVAL, "lk_rms_norm_i8: dtype and gain_dtype are LK_F32, LK_F16 or LK_BF16");
    if (rows < 0 || dim < 1) return fail(LK_EINVAL, "lk_rms_norm_i8: bad size");
    if (dim > LK_NORM_MAX_DIM) return fail(LK_ERANGE, "lk_rms_norm_i8: dim is limited to LK_NORM_MAX_DIM (32768)");
    if (rows > 0x7fffffff) return fail(LK_ERANGE, "lk_rms_norm_i8: more than 2^31-1 rows");
    if (!(eps >= 0.0f && eps <= FLT_MAX)) return fail(LK_EINVAL, "lk_rms_norm_i8: eps must be finite and not negative");
    if (rows > 0 && (!d_x || !d_codes || !d_scales)) return fail(LK_EINVAL, "lk_rms_norm_i8: NULL pointer");
    if (rows > 1 && (ldx < dim || ldc < dim || (d_residual && ldr < dim) || (d_sum && lds < dim)))
        return fail(LK_EINVAL, "lk_rms_norm_i8: a row stride is smaller than dim");
    const int eb = type_bytes(dtype);
    const uintptr_t mask = (uintptr_t)eb - 1;
    if ((reinterpret_cast<uintptr_t>(d_x) & mask) || (reinterpret_cast<uintptr_t>(d_residual) & mask) ||
        (reinterpret_cast<uintptr_t>(d_sum) & mask) || (d_gain && reinterpret_cast<uintptr_t>(d_gain) % type_bytes(gain_dtype)) ||
        (reinterpret_cast<uintptr_t>(d_scales) & 3))
        return fail(LK_EINVAL, "lk_rms_norm_i8: a pointer is not aligned to its element type");
    DeviceScope scope;
    LK_TRY(scope.enter(device, "lk_rms_norm_i8"));
    if (rows == 0) return LK_OK;
    NormArgs a = {d_x, d_residual, d_gain, d_sum, reinterpret_cast<signed char *>(d_codes), d_scales,
                  rows, ldx, ldr, lds, ldc, dim, gain_dtype, eps};
    const bool vec = aligned_rows(d_x, ldx, eb, 16) && (!d_residual || aligned_rows(d_residual, ldr, eb, 16)) &&
                     (!d_sum || aligned_rows(d_sum, lds, eb, 16)) && aligned_rows(d_codes, ldc, 1, 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == LK_F32) return vec ? norm_launch<float, true>(a, st) : norm_launch<float, false>(a, st);
    if (dtype == LK_F16) return vec ? norm_launch<__half, true>(a, st) : norm_launch<__half, false>(a, st);
    return vec ? norm_launch<__nv_bfloat16, true>(a, st) : norm_launch<__nv_bfloat16, false>(a, st);
}
