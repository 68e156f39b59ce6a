// Root-mean-square norm of x (+ residual) with an int8 output, one scale per row.
//
//   h = x + r;  y = h * inv * g with inv = 1 / sqrt(mean(h^2) + eps);  s = max|y| / 127;  c = round(y / s)
//
// inv is one positive number per row, so with p = h * g:  max|y| = inv * max|p| and y / s = 127 p / max|p|.
// The codes do not need inv at all, and both reductions of a row (the sum of h^2 and the maximum of
// |p|) are taken in ONE meeting of its threads, from values that stay in registers: x and r are read once,
// the sum and the codes written once.  The maximum, which every thread needs, is one of bit patterns (ordered like the
// values, NaN above infinity); the sum goes to the first warp alone, which takes the row's one square root.  It is a float64
// sum: float32 squares overflow from |h| = 1.8e19 on, and a row's sum is then the same to the last bits in any order.
//
// Bound: HBM (x, r and the sum at their types, one byte of code per element).  Two kernels:
// * k_norm_rows, many rows: a CTA streams rows through a ring of shared-memory stages filled by bulk copies, so the bytes in
//   flight do not depend on registers; the gain stays in registers.
// * k_norm_row, few rows, rows off 16-byte boundaries or too wide for a stage: a CTA per row, loads straight to registers.
// Conversions issue on a narrow pipe (16 lanes per clock and SM), so a code is rounded by adding 1.5 * 2^23, which leaves it
// in the low byte, and not by two conversions; one per element is left, the widening for the sum.
#include <cfloat>
#include <type_traits>

#include "devops.cuh"
#include "tensor5.cuh"

namespace lk {

struct NormArgs {
    const void *x, *r, *gain;
    void *sum;
    signed char *codes;
    float *scales;
    long long rows, ldx, ldr, lds, ldc;
    int dim, gain_type, gain_vec;
    float eps;
    double per_dim;  // 1 / dim
    int stages, stage_bytes, row_bytes;
};

static __device__ unsigned g_norm_failed;  // a bounded wait ran out on this device

constexpr unsigned kInfBits = 0x7f800000u;

template <int THREADS>
struct NormShared {
    double sums[2][THREADS];                 // every thread's sum of squares, and every warp's max|p|: of this row and
    alignas(16) unsigned tops[2][THREADS / 32 < 4 ? 4 : THREADS / 32];  // the one before, which one warp may still be at
    unsigned long long full[16];
    int slow;                                // some row is one for slow_row
    int failed[2];                           // a wait for this row, or the one before, ran out
};

struct Raw {
    unsigned q[8];  // eight elements as they lie in memory (16-bit types: the first four words alone)
};
template <typename T>
__device__ __forceinline__ void unpack(const Raw &w, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w.q[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w.q[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w.q[i] << 16), v[2 * i + 1] = __uint_as_float(w.q[i] & 0xffff0000u);
    }
}
template <typename T>
__device__ __forceinline__ void pack(const float (&v)[8], Raw &w) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w.q[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<__half2 *>(&w.q[i]) = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<__nv_bfloat162 *>(&w.q[i]) = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    }
}
// max(|a|, |b|, |c|), NaN if any of them is
__device__ __forceinline__ float top3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A row that is not finite, or where h * g leaves the comfortable range of float32 (overflow, or max|p| below 2^-100, 0 among that
// where h is not all 0): all of it again in float64, from memory.
template <typename T, int THREADS>
__device__ void slow_row(const NormArgs &a, NormShared<THREADS> &s, long long row) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx, *r = static_cast<const T *>(a.r) + row * a.ldr;
    const auto sum_of = [&](int e) {
        const float h = Elem<T>::get(x[e]);
        return a.r != nullptr ? h + Elem<T>::get(r[e]) : h;
    };
    const auto product = [&](float h, int e) { return (double)h * (a.gain != nullptr ? (double)load_as(a.gain_type, a.gain, e) : 1.0); };
    double top = 0.0, ss = 0.0;
#pragma unroll 1
    for (int e = tid; e < a.dim; e += THREADS) {
        const float h = sum_of(e);
        const double q = fabs(product(h, e));
        ss = fma((double)h, (double)h, ss);
        top = q < CUDART_INF ? fmax(top, q) : CUDART_INF;  // NaN too: nothing comes back from there
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    __syncthreads();
    if (lane == 0) s.sums[0][warp] = ss, s.sums[1][warp] = top;
    __syncthreads();
    ss = 0.0;
#pragma unroll 1
    for (int w = 0; w < THREADS / 32; ++w) ss += s.sums[0][w], top = fmax(top, s.sums[1][w]);
    float scale = (float)(top * rsqrt(ss * a.per_dim + (double)a.eps) / 127.0);
    const bool good = top < CUDART_INF && ss < CUDART_INF && scale < CUDART_INF_F;
    if (!good) scale = CUDART_NAN_F;
    const double step = good && top > 0.0 ? 127.0 / top : 0.0;  // gains of zero alone: codes and scale are 0
#pragma unroll 1
    for (int e = tid; e < a.dim; e += THREADS) {
        const float h = sum_of(e);  // before its place is written: x or r may be where the sum goes
        a.codes[row * a.ldc + e] = good ? (signed char)(int)rint(fmin(fmax(product(h, e) * step, -127.0), 127.0)) : (signed char)0;
        if (a.sum != nullptr) static_cast<T *>(a.sum)[row * a.lds + e] = Elem<T>::put(h);
    }
    if (tid == 0) a.scales[row] = scale;
}

// The threads of a CTA on one row.  A thread holds V groups of eight elements: consecutive ones read by 16-byte loads (VEC), or
// element e of the row belongs to thread e % THREADS.
template <typename T, int THREADS, int V, bool VEC>
struct NormRow {
    static constexpr int WARPS = THREADS / 32;
    const NormArgs &a;
    NormShared<THREADS> &s;
    const int tid, lane, warp;
    __device__ __forceinline__ int at(int v, int i) const { return VEC ? (v * THREADS + tid) * 8 + i : (v * 8 + i) * THREADS + tid; }
    __device__ __forceinline__ bool whole(int v) const { return VEC && at(v, 0) + 8 <= a.dim; }

    template <typename E>
    __device__ __forceinline__ void fetch(const E *from, int v, bool wide_loads, Raw &w) const {
        if (wide_loads && whole(v)) {
            const uint4 p = *reinterpret_cast<const uint4 *>(from + at(v, 0));
            w.q[0] = p.x, w.q[1] = p.y, w.q[2] = p.z, w.q[3] = p.w;
            if (sizeof(E) == 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(from + at(v, 4));
                w.q[4] = o.x, w.q[5] = o.y, w.q[6] = o.z, w.q[7] = o.w;
            }
        } else {
            unsigned e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = 0u;
                if (at(v, i) < a.dim) e[i] = sizeof(E) == 4 ? reinterpret_cast<const unsigned *>(from)[at(v, i)] : reinterpret_cast<const unsigned short *>(from)[at(v, i)];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (sizeof(E) == 4) w.q[i] = e[i];
                else if (i < 4) w.q[i] = e[2 * i] | e[2 * i + 1] << 16;
            }
        }
    }
    __device__ __forceinline__ void gain_of(int v, float (&g)[8]) const {
        Raw w = {};
        if (a.gain == nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = 1.0f;
        } else if (a.gain_type == LK_F32) {
            fetch(static_cast<const float *>(a.gain), v, a.gain_vec, w);
            unpack<float>(w, g);
        } else {
            fetch(static_cast<const __half *>(a.gain), v, a.gain_vec, w);
            if (a.gain_type == LK_F16) unpack<__half>(w, g);
            else unpack<__nv_bfloat16>(w, g);
        }
    }

    // From the row's raw x, r and gain to its outputs; true, and nothing written, where it is one for slow_row.  `met` runs
    // once behind the meeting of the threads, when the raw values have been used.
    template <typename F>
    __device__ __forceinline__ bool finish(long long row, int round, const Raw (&xw)[V], const Raw (&rw)[V], const float (&g)[V][8], F met) const {
        const int turn = round & 1;
        T *sum = static_cast<T *>(a.sum) + row * a.lds;
        signed char *codes = a.codes + row * a.ldc;
        float p[V][8];
        Raw rounded[V];  // h as it will be stored: the store waits, so that x and r, which may be where it goes, can be read again
        double ss = 0.0, ss2 = 0.0;
        float high = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float h[8];
            unpack<T>(xw[v], h);
            if (a.r != nullptr) {
                float rv[8];
                unpack<T>(rw[v], rv);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] += rv[i];
            }
            pack<T>(h, rounded[v]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i & 1) ss2 = fma((double)h[i], (double)h[i], ss2);
                else ss = fma((double)h[i], (double)h[i], ss);
                p[v][i] = h[i] * g[v][i];
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) high = top3(high, p[v][i], p[v][i + 1]);
        }
        unsigned top = __float_as_uint(high) & 0x7fffffffu;
        if (top == 0u && ss + ss2 != 0.0) top = 1u;  // h is not zero here: a product that underflowed, or a gain of zero (slow_row tells)
        top = __reduce_max_sync(0xffffffffu, top);
        s.sums[turn][tid] = ss + ss2;
        if (lane == 0) s.tops[turn][warp] = top;
        if (WARPS > 1) __syncthreads();
        else __syncwarp();
        met();
        if constexpr (WARPS % 4 == 0) {
#pragma unroll
            for (int w = 0; w < WARPS; w += 4) {
                const uint4 q = *reinterpret_cast<const uint4 *>(&s.tops[turn][w]);
                top = max(max(max(top, q.x), max(q.y, q.z)), q.w);
            }
        }
        float step = 0.0f;  // of a row of nothing but zeros
        if (top >= kInfBits || (top != 0u && top < 0x0d800000u)) return true;  // all threads agree
        if (top != 0u) step = 127.0f / __uint_as_float(top);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unsigned c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)  // |p step| <= 127 (1 + 2^-23): rounds to 127 at most
                c[i] = __float_as_uint(fmaf(p[v][i], step, 12582912.0f));
            const uint2 q = {__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                             __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410)};
            if (whole(v)) {
                if (a.sum != nullptr) {
                    const unsigned(&w)[8] = rounded[v].q;
                    *reinterpret_cast<uint4 *>(sum + at(v, 0)) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(sum + at(v, 4)) = make_uint4(w[4], w[5], w[6], w[7]);
                }
                *reinterpret_cast<uint2 *>(codes + at(v, 0)) = q;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at(v, i) < a.dim) {
                        if (a.sum != nullptr) {
                            if (sizeof(T) == 4) reinterpret_cast<unsigned *>(sum)[at(v, i)] = rounded[v].q[i];
                            else reinterpret_cast<unsigned short *>(sum)[at(v, i)] = (unsigned short)(rounded[v].q[i / 2] >> (16 * (i & 1)));
                        }
                        codes[at(v, i)] = (signed char)((i < 4 ? q.x >> (8 * i) : q.y >> (8 * i - 32)) & 0xffu);
                    }
            }
        }
        // The sum of squares and the row's square root: one warp's work, another one's for the next row, under the others' way
        // to the next meeting.
        bool over = false;
        if (warp == round % WARPS) {
            ss = 0.0;
#pragma unroll
            for (int t = 0; t < THREADS; t += 32) ss += s.sums[turn][t + lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (lane == 0) {
                float scale = 0.0f;  // a row of zeros: 0, whatever eps is
                if (top != 0u) {
                    const double y = (double)__uint_as_float(top) * rsqrt(ss * a.per_dim + (double)a.eps);
                    scale = (float)y / 127.0f;
                    if (!(scale < CUDART_INF_F)) scale = (float)(y / 127.0);  // a y past float32 may have a scale that is not
                    if (!(scale < CUDART_INF_F)) scale = CUDART_NAN_F, over = true;
                }
                a.scales[row] = scale;
            }
        }
        // A scale is at most sqrt(dim) / 127 times the largest gain, so only a row wider than 127^2 can have one past float32.
        if constexpr (THREADS * V * 8 > 127 * 127) {
            if (__syncthreads_or(over))
#pragma unroll 1
                for (int e = tid; e < a.dim; e += THREADS) codes[e] = 0;
        }
        return false;
    }
};

template <typename T, int THREADS, int V, bool VEC>
__global__ void __launch_bounds__(THREADS, 1) k_norm_row(const __grid_constant__ NormArgs a) {
    __shared__ NormShared<THREADS> s;
    using Row = NormRow<T, THREADS, V, VEC>;
    const Row w = {a, s, (int)threadIdx.x, (int)threadIdx.x & 31, (int)threadIdx.x >> 5};
    const long long row = blockIdx.x;
    Raw xw[V] = {}, rw[V] = {};
    float g[V][8];
    const T *x = static_cast<const T *>(a.x) + row * a.ldx, *r = static_cast<const T *>(a.r) + row * a.ldr;
#pragma unroll
    for (int v = 0; v < V; ++v) w.fetch(x, v, true, xw[v]);
    if (a.r != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) w.fetch(r, v, true, rw[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) w.gain_of(v, g[v]);
    if (w.finish(row, 0, xw, rw, g, [] {})) slow_row<T, THREADS>(a, s, row);
}

// Rows blockIdx.x, + gridDim.x, ... through a ring of stages, each a row of x and one of r.
template <typename T, int THREADS, int V, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) k_norm_rows(const __grid_constant__ NormArgs a) {
    extern __shared__ __align__(128) unsigned char n_raw[];
    using Shared = NormShared<THREADS>;
    Shared &s = *reinterpret_cast<Shared *>(n_raw);
    unsigned char *ring = n_raw + (sizeof(Shared) + 127) / 128 * 128;
    using Row = NormRow<T, THREADS, V, true>;
    const Row w = {a, s, (int)threadIdx.x, (int)threadIdx.x & 31, (int)threadIdx.x >> 5};
    const int half = a.stage_bytes / 2;  // where r's row starts
    const auto ask = [&](long long row, int stage) {  // one thread
        const unsigned bytes = (unsigned)a.row_bytes * (a.r != nullptr ? 2u : 1u);
        g_mbar_expect_tx(&s.full[stage], bytes);
        const auto copy = [&](const void *from, unsigned char *to) {
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(g_smem(to)), "l"(from),
                         "r"((unsigned)a.row_bytes), "r"(g_smem(&s.full[stage]))
                         : "memory");
        };
        copy(static_cast<const T *>(a.x) + row * a.ldx, ring + (size_t)stage * a.stage_bytes);
        if (a.r != nullptr) copy(static_cast<const T *>(a.r) + row * a.ldr, ring + (size_t)stage * a.stage_bytes + half);
    };
    if (w.tid == 0) {
        for (int i = 0; i < a.stages; ++i) g_mbar_init(&s.full[i], 1);
        s.failed[0] = s.failed[1] = s.slow = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < a.stages && blockIdx.x + (long long)i * gridDim.x < a.rows; ++i) ask(blockIdx.x + (long long)i * gridDim.x, i);
    }
    float g[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) w.gain_of(v, g[v]);
    __syncthreads();
    int stage = 0;
    unsigned phase = 0, round = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, ++round) {
        g_mbar_wait(&s.full[stage], phase, &s.failed[round & 1]);
        const T *x = reinterpret_cast<const T *>(ring + (size_t)stage * a.stage_bytes);
        const T *r = reinterpret_cast<const T *>(ring + (size_t)stage * a.stage_bytes + half);
        Raw xw[V] = {}, rw[V] = {};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            w.fetch(x, v, true, xw[v]);
            if (a.r != nullptr) w.fetch(r, v, true, rw[v]);
        }
        bool failed = false;
        const bool slow = w.finish(row, (int)round, xw, rw, g, [&] {  // all threads have the row in registers: its stage is free
            const long long next = row + (long long)a.stages * gridDim.x;
            failed = *(volatile int *)&s.failed[round & 1] != 0;  // set, if at all, before the meeting
            if (w.tid == 0 && next < a.rows && !failed) ask(next, stage);
        });
        if (failed) break;
        if (slow && w.tid == 0) a.scales[row] = -1.0f, s.slow = 1;  // marked: its turn comes behind the others
        if (++stage == a.stages) stage = 0, phase ^= 1u;
    }
    __syncthreads();
    if (s.slow != 0)
        for (long long row = blockIdx.x; row < a.rows; row += gridDim.x)
            if (*(volatile float *)(a.scales + row) == -1.0f) slow_row<T, THREADS>(a, s, row);
    if ((s.failed[0] | s.failed[1]) != 0) {
        if (w.tid == 0) atomicExch(&g_norm_failed, 1u);
        const long long t0 = clock64();  // copies may still be landing in this CTA's shared memory
        while (clock64() - t0 < 2000000ll) {}
    }
}

template <typename T, bool VEC>
static int row_launch(const NormArgs &a, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    const int groups = (a.dim + 7) / 8;
    const char *who = "lk_rms_norm_i8";
    if (groups <= 32) return launch(who, k_norm_row<T, 32, 1, VEC>, grid, 32, st, a);
    if (groups <= 128) return launch(who, k_norm_row<T, 128, 1, VEC>, grid, 128, st, a);
    if (groups <= 512) return launch(who, k_norm_row<T, 256, 2, VEC>, grid, 256, st, a);
    if (groups <= 1024) return launch(who, k_norm_row<T, 512, 2, VEC>, grid, 512, st, a);
    return launch(who, k_norm_row<T, 1024, 4, VEC>, grid, 1024, st, a);
}

// Rows in a CTA's ring, and the launch; -1 where the other kernel is the one to take.
template <typename T, int THREADS, int V, int PER_SM>
static int rows_launch(NormArgs a, int device, cudaStream_t st) {
    static OncePerDevice sized;
    const int fixed = (int)(sizeof(NormShared<THREADS>) + 127) / 128 * 128;
    const int part = (a.row_bytes + 127) / 128 * 128;
    a.stage_bytes = 2 * part;
    a.stages = std::min((227 * 1024 / PER_SM - 1024 - fixed) / a.stage_bytes, 16);
    if (a.stages < 2) return -1;
    LK_TRY(sized.run(device, [] {
        LK_CUDA(cudaFuncSetAttribute((const void *)k_norm_rows<T, THREADS, V, PER_SM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        return 0;
    }));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<long long>(a.rows, (long long)sm_count(device) * PER_SM));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)fixed + (size_t)a.stages * a.stage_bytes;
    cfg.stream = st;
    return launch_cfg("lk_rms_norm_i8", k_norm_rows<T, THREADS, V, PER_SM>, cfg, a);
}

template <typename T>
static int norm_launch(const NormArgs &a, bool vec, int device, cudaStream_t st) {
    if (!vec) return row_launch<T, false>(a, st);
    if (a.row_bytes % 16 == 0 && a.rows >= 4ll * sm_count(device) && a.dim > 256) {
        const int groups = (a.dim + 7) / 8;
        int r = -1;
        if (groups <= 128) r = rows_launch<T, 128, 1, 6>(a, device, st);
        else if (groups <= 256) r = rows_launch<T, 256, 1, 4>(a, device, st);
        else if (groups <= 512) r = rows_launch<T, 256, 2, 3>(a, device, st);
        else if (groups <= 1024) r = rows_launch<T, 512, 2, 2>(a, device, st);
        if (r >= 0) return r;
    }
    return row_launch<T, true>(a, st);
}

// Whether a wait ran out on the current device since the last call; the flag is lowered.
int norm_failed(int *out) {
    unsigned v = 0, zero = 0;
    LK_CUDA(cudaMemcpyFromSymbol(&v, g_norm_failed, sizeof v));
    if (v) LK_CUDA(cudaMemcpyToSymbol(g_norm_failed, &zero, sizeof zero));
    *out = v != 0;
    return 0;
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
                  rows, ldx, ldr, lds, ldc, dim, gain_dtype, d_gain && reinterpret_cast<uintptr_t>(d_gain) % 16 == 0, eps, 1.0 / dim,
                  0, 0, dim * eb};
    const bool vec = aligned_rows(d_x, ldx, eb, 16) && (!d_residual || aligned_rows(d_residual, ldr, eb, 16)) &&
                     (!d_sum || aligned_rows(d_sum, lds, eb, 16)) && aligned_rows(d_codes, ldc, 1, 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == LK_F32) return norm_launch<float>(a, vec, device, st);
    if (dtype == LK_F16) return norm_launch<__half>(a, vec, device, st);
    return norm_launch<__nv_bfloat16>(a, vec, device, st);
}
