// One draw per row of scores: temperature, top-k, top-p, min-p, from given random numbers.
//
// Every filter keeps a prefix of the row's order (score descending, index ascending), so what is kept is
// described by one score X and a number of ties: all scores above X, and the first `ties` entries (by
// index) that equal it.  No sort is needed: X is found by bisection over the order-preserving image of
// the scores, with counts (top-k) or weights (top-p) of the entries at or above a trial value.
//
// Weights w = exp((x - max) / T) are computed in float64 and summed as 64-bit integers, w * 2^F with
// vocab * 2^F <= 2^63: sums do not depend on their order, the prefix that a cut finds and the running
// sum that a draw walks agree to the last bit, and a border between two entries is met to ~2^-44 of the
// largest weight.
//
// One CTA per row; passes over the row after the first come from L2.
#include "devops.cuh"

namespace lk {

struct SampleArgs {
    const void *logits;
    long long ld;
    int vocab;
    const float *temperature, *top_p, *min_p, *u;
    const int *top_k;
    long long *ids;
    float *probs;
    int *kept;
    double unit;  // 2^F
};

constexpr unsigned kNegInf = 0x007fffffu;  // image of -infinity; NaN (0) is below it
constexpr int ST = 1024;

struct SampleShared {
    unsigned long long sum[32];
    unsigned top[32];
    unsigned long long total;
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long block_sum(SampleShared &s, unsigned long long v) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long t = 0;
#pragma unroll
    for (int w = 0; w < ST / 32; ++w) t += s.sum[w];
    return t;
}

template <typename T>
__global__ void __launch_bounds__(ST) k_sample(const SampleArgs a) {
    __shared__ SampleShared s;
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = a.vocab;

    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float least = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;  // the first is always kept
    const float u = a.u[row];
    const bool bad = !(temp >= 0.0f) || p != p || (a.min_p && a.min_p[row] != a.min_p[row]) || u != u;
    if (temp == 0.0f) temp = 1.0f, k = 1;

    unsigned top = 0;
    unsigned long long valid = 0;
    for (int i = tid; i < vocab; i += ST) {
        const unsigned o = ord_from_f32(Elem<T>::get(x[i]));
        top = max(top, o);
        valid += o > kNegInf;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s.top[warp] = top;
    valid = block_sum(s, valid);
#pragma unroll
    for (int w = 0; w < ST / 32; ++w) top = max(top, s.top[w]);
    if (bad || valid == 0) {
        if (tid == 0) {
            a.ids[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
            if (a.kept) a.kept[row] = 0;
        }
        return;
    }
    const double x_top = (double)f32_from_ord(top), per_t = 1.0 / (double)temp;
    const auto weight = [&](unsigned o) -> double {
        return o == top ? 1.0 : exp(((double)f32_from_ord(o) - x_top) * per_t);
    };
    const auto weight_int = [&](unsigned o) { return (unsigned long long)__double2ull_rn(weight(o) * a.unit); };

    unsigned cut = kNegInf + 1;             // kept: images above `cut`, and the first `ties` equal to it
    unsigned long long ties = ~0ull;
    if (k > 0 && (unsigned long long)k < valid) {
        unsigned lo = kNegInf + 1, hi = top;  // count(>= lo) >= k; the largest such value
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo + 1) / 2;
            unsigned long long c = 0;
            for (int i = tid; i < vocab; i += ST) c += ord_from_f32(Elem<T>::get(x[i])) >= mid;
            c = block_sum(s, c);
            if (c >= (unsigned long long)k) lo = mid; else hi = mid - 1;
        }
        unsigned long long above = 0;
        for (int i = tid; i < vocab; i += ST) above += ord_from_f32(Elem<T>::get(x[i])) > lo;
        cut = lo, ties = k - block_sum(s, above);
    }
    if (p < 1.0f) {
        // weight of the prefix at or above `from` (the ties of `cut` counted by number: they weigh the same)
        const auto mass = [&](unsigned from, bool with_from) {
            unsigned long long m = 0, eq = 0;
            for (int i = tid; i < vocab; i += ST) {
                const unsigned o = ord_from_f32(Elem<T>::get(x[i]));
                if (o > cut && (o > from || (with_from && o == from))) m += weight_int(o);
                eq += o == cut;
            }
            m = block_sum(s, m);
            eq = block_sum(s, eq);
            if (cut > from || (with_from && cut == from)) m += min(eq, ties) * weight_int(cut);
            return m;
        };
        const unsigned long long all = mass(cut, true);
        const unsigned long long want = p <= 0.0f ? 0ull : (unsigned long long)ceil((double)p * (double)all);
        unsigned lo = cut, hi = top;  // mass(>= lo) >= want; the largest such value
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo + 1) / 2;
            if (mass(mid, true) >= want) lo = mid; else hi = mid - 1;
        }
        const unsigned long long before = mass(lo, false), each = weight_int(lo);
        unsigned long long need = before >= want ? 0ull : (each ? (want - before + each - 1) / each : ~0ull);
        if (lo == top && need == 0) need = 1;
        if (lo == cut) need = min(need, ties);
        cut = lo, ties = need;
    }

    // The kept weights in the order of the indexes: thread t owns entries t + ST * j, so a warp's turn is 32
    // consecutive entries and a CTA's 1,024.  First their sum and number, then the walk to the draw.
    for (int walk = 0; walk < 2; ++walk) {
        __shared__ unsigned long long target;
        unsigned long long run = 0, seen = 0;  // weight and ties of all turns so far
        unsigned long long count = 0;
        for (int i0 = 0; i0 < vocab; i0 += ST) {
            const int i = i0 + tid;
            const unsigned o = i < vocab ? ord_from_f32(Elem<T>::get(x[i])) : 0u;
            // place among the ties
            const unsigned eq = __ballot_sync(0xffffffffu, o == cut);
            __syncthreads();
            if (lane == 0) s.sum[warp] = __popc(eq);
            __syncthreads();
            unsigned long long place = seen + __popc(eq & lanemask_lt());
            for (int w = 0; w < ST / 32; ++w) {
                if (w < warp) place += s.sum[w];
                seen += s.sum[w];
            }
            const double w = weight(o);
            const bool keep = (o > cut || (o == cut && place < ties)) && (least <= 0.0f || w >= (double)least);
            const unsigned long long mine = keep ? (unsigned long long)__double2ull_rn(w * a.unit) : 0ull;
            count += keep;
            unsigned long long inc = mine;  // running sum within the turn
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned long long v = shfl_up_u64(inc, d);
                if (lane >= d) inc += v;
            }
            __syncthreads();
            if (lane == 31) s.sum[warp] = inc;
            __syncthreads();
            unsigned long long base = run;
            for (int w2 = 0; w2 < ST / 32; ++w2) {
                if (w2 < warp) base += s.sum[w2];
                run += s.sum[w2];
            }
            if (walk == 1 && base + inc - mine <= target && target < base + inc) {  // one entry of the row
                a.ids[row] = i;
                if (a.probs) a.probs[row] = (float)((double)mine / (double)s.total);
            }
        }
        if (walk == 0) {
            count = block_sum(s, count);
            __syncthreads();
            if (tid == 0) {
                s.total = run;
                const double t = (double)u * (double)run;
                target = t <= 0.0 ? 0ull : (t >= (double)run ? run - 1 : min((unsigned long long)t, run - 1));
                if (a.kept) a.kept[row] = (int)count;
            }
            __syncthreads();
        }
    }
}

template <typename T>
static int sample_launch(const SampleArgs &a, long long rows, cudaStream_t st) {
    return launch("lk_sample", k_sample<T>, (unsigned)rows, ST, st, a);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_sample(int device, int dtype, int64_t rows, int64_t vocab, const void *d_logits, int64_t ld,
                         const float *d_temperature, const int32_t *d_top_k, const float *d_top_p, const float *d_min_p,
                         const float *d_u, int64_t *d_ids, float *d_probs, int32_t *d_kept, void *stream) {
    if (!float_type(dtype)) return fail(LK_EINVAL, "lk_sample: dtype is LK_F32, LK_F16 or LK_BF16");
    if (rows < 0 || vocab < 0) return fail(LK_EINVAL, "lk_sample: bad size");
    if (vocab > LK_SAMPLE_MAX_VOCAB) return fail(LK_ERANGE, "lk_sample: vocab is limited to LK_SAMPLE_MAX_VOCAB (16777216)");
    if (rows > 0x7fffffff) return fail(LK_ERANGE, "lk_sample: more than 2^31-1 rows");
    if (rows > 0 && ((vocab > 0 && !d_logits) || !d_u || !d_ids)) return fail(LK_EINVAL, "lk_sample: NULL pointer");
    if (rows > 1 && ld < vocab) return fail(LK_EINVAL, "lk_sample: the row stride is smaller than vocab");
    const auto off = [](const void *p, int to) { return reinterpret_cast<uintptr_t>(p) % to != 0; };
    if (off(d_logits, type_bytes(dtype)) || off(d_temperature, 4) || off(d_top_k, 4) || off(d_top_p, 4) || off(d_min_p, 4) ||
        off(d_u, 4) || off(d_ids, 8) || off(d_probs, 4) || off(d_kept, 4))
        return fail(LK_EINVAL, "lk_sample: a pointer is not aligned to its element type");
    DeviceScope scope;
    LK_TRY(scope.enter(device, "lk_sample"));
    if (rows == 0) return LK_OK;
    int bits = 0;  // 2^bits >= vocab
    while ((1ll << bits) < vocab) ++bits;
    SampleArgs a = {d_logits, ld, (int)vocab, d_temperature, d_top_p, d_min_p, d_u, d_top_k,
                    reinterpret_cast<long long *>(d_ids), d_probs, d_kept, (double)(1ull << (63 - bits))};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == LK_F32) return sample_launch<float>(a, rows, st);
    if (dtype == LK_F16) return sample_launch<__half>(a, rows, st);
    return sample_launch<__nv_bfloat16>(a, rows, st);
}
