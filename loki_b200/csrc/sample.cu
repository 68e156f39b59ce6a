// One draw per row of scores: temperature, top-k, top-p, min-p, from given random numbers.
//
// Every filter keeps a prefix of the row's order (score descending, index ascending), so what is kept is
// described by its last entry: a 64-bit ranking key (score image, ~index) at or above which entries are kept.  No
// sort is needed; a cut is found by histograms over the order, with counts (top-k) or weights (top-p).
//
// Weights w = exp((x - max) / T) are computed in float64 and summed as 64-bit integers, w * 2^F with
// vocab * 2^F <= 2^63: sums do not depend on their order (shared-memory atomics, warps, CTAs), the prefix that a
// cut finds and the running sum that a draw walks agree to the last bit, and a border between two entries
// is met to ~2^-44 of the largest weight.
//
// A cluster of CTAs owns a row.  Each loads one stretch of it into its shared memory (what does not fit is read
// again from L2), so scores cross HBM once; every later pass runs over shared memory, and the CTAs
// exchange maxima, histograms and sums through distributed shared memory.
//
// A cut: entries fall into 1,024 bins by the distance d = max - x, 32 bins to a factor of two (the image
// of d without its low bits: monotone in x, and fine where a softmax has its weight).  The bin in which the
// measure reaches its target is cut again: up to 1,024 entries are gathered in one CTA, where each counts
// what ranks above it; more are binned again by their images; entries that are all equal are cut by index.
#include "devops.cuh"

namespace lk {

struct SampleArgs {
    const void *logits;
    long long ld;
    int vocab;
    int ctas, seg, cap;  // CTAs per row, entries per CTA, how many of those its shared memory holds
    const float *temperature, *top_p, *min_p, *u;
    const int *top_k;
    long long *ids;
    float *probs;
    int *kept;
    double unit;  // 2^F
};

constexpr unsigned kNegInf = 0x007fffffu;  // image of -infinity; NaN (0) is below it
constexpr int ST = 1024, SWARPS = ST / 32;
constexpr int SBINS = 1024;
constexpr int SLIST = 1024;
constexpr int SMAX_CTAS = 16;
using u64 = unsigned long long;

struct alignas(16) SampleShared {
    unsigned lo[SBINS], hi[SBINS], n[SBINS];   // this CTA's bins: weights (two words), entries
    u64 all_w[SBINS];                          // the row's bins
    unsigned all_n[SBINS];
    u64 list[SLIST];                           // the leader's: keys of the bin being cut
    u64 warp_w[SWARPS];
    unsigned warp_n[SWARPS];
    u64 slot_w[SMAX_CTAS];                     // one word from every CTA of the row
    unsigned slot_a[SMAX_CTAS], slot_b[SMAX_CTAS];
    unsigned listed;
    u64 cut;                                   // a decision of the leader or of the CTA that holds an entry
    u64 found_w, found_before;
    int found;
};

__device__ __forceinline__ unsigned s_at(const void *p, int rank) {  // a shared-memory address as it sits in CTA `rank`
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void s_put(unsigned at, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void s_put(unsigned at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ unsigned s_get(unsigned at) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned s_add(unsigned at, unsigned v) {
    unsigned old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
    return old;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const u64 o = shfl_up_u64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// One row, as the CTAs of its cluster see it.
template <typename T>
struct Row {
    const SampleArgs &a;
    SampleShared &s;
    T *data;        // this CTA's stretch in shared memory, `cap` entries of it
    const T *x;     // the row
    int rank, start, len, wlen, tid, lane, warp;
    unsigned top;
    double x_top, per_t;
    u64 thr;        // entries with a key at or above this are kept

    __device__ __forceinline__ void sync() const {
        if (a.ctas > 1) {
            asm volatile("barrier.cluster.arrive;" ::: "memory");
            asm volatile("barrier.cluster.wait;" ::: "memory");
        } else
            __syncthreads();
    }
    __device__ __forceinline__ unsigned image(int i) const { return ord_from_f32(Elem<T>::get(i < a.cap ? data[i] : x[start + i])); }
    __device__ __forceinline__ double weight(unsigned o) const {
        return o == top ? 1.0 : exp(((double)f32_from_ord(o) - x_top) * per_t);
    }
    __device__ __forceinline__ u64 whole(double w) const { return __double2ull_rn(w * a.unit); }
    __device__ __forceinline__ u64 key(unsigned o, int i) const { return make_key(o, (unsigned)(start + i)); }

    // f(image, local index) for every entry of this warp; lanes past the end see image 0 (never kept)
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int lo = warp * wlen, hi = min(lo + wlen, len);
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            f(i < hi ? image(i) : 0u, i);
        }
    }

    // Sum of f over the row, by integers; warp_w keeps this CTA's warps' sums and slot_w the CTAs'.
    template <typename F>
    __device__ u64 sums(F f) const {
        u64 w = 0;
        each([&](unsigned o, int i) { w += f(o, i); });
        w = warp_sum(w);
        __syncthreads();
        if (lane == 0) s.warp_w[warp] = w;
        __syncthreads();
        if (warp == 0) {
            w = warp_sum(s.warp_w[lane]);
            if (lane < a.ctas) s_put(s_at(&s.slot_w[rank], lane), w);
        }
        sync();
        u64 all = 0;
        for (int r = 0; r < a.ctas; ++r) all += s.slot_w[r];
        return all;
    }
    // The entry at which the running sum of f (in the order of the indexes) first exceeds `target`, which
    // is below the sum that sums(f) has just returned: the CTA that holds it sets found (local index),
    // found_w (its f) and found_before; in the others found is -1.  No meeting of the cluster.
    template <typename F>
    __device__ void walk(F f, u64 target) const {
        __syncthreads();
        if (tid == 0) s.found = -1;
        u64 before = 0;
        for (int r = 0; r < rank; ++r) before += s.slot_w[r];
        const bool mine = before <= target && target < before + s.slot_w[rank];
        __syncthreads();
        if (!mine) return;
        int lo = 0, n = wlen;  // first the stretch of a warp, then a 32nd of that, then its entries
        for (int level = 0;; ++level) {
            int at = 0;
            u64 run = before;
            for (; at < SWARPS - 1 && run + s.warp_w[at] <= target; ++at) run += s.warp_w[at];
            before = run;
            lo += at * n;
            if (level == 1) break;
            const int end = min(lo + n, len);
            n = ((n + SWARPS - 1) / SWARPS + 31) & ~31;
            u64 w = 0;
            for (int i0 = lo + warp * n; i0 < min(lo + (warp + 1) * n, end); i0 += 32) {
                const int i = i0 + lane;
                if (i < end) w += f(image(i), i);
            }
            w = warp_sum(w);
            __syncthreads();
            if (lane == 0) s.warp_w[warp] = w;
            __syncthreads();
        }
        if (warp == 0) {
            for (int i0 = lo; i0 < min(lo + n, len); i0 += 32) {
                const int i = i0 + lane;
                const u64 w = i < len ? f(image(i), i) : 0ull;
                const u64 inc = warp_scan(w, lane) + before;
                const unsigned past = __ballot_sync(0xffffffffu, inc > target);
                if (past) {
                    if (lane == __ffs(past) - 1) s.found = i, s.found_w = w, s.found_before = inc - w;
                    break;
                }
                before = __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        __syncthreads();
    }

    // The bin of an entry: by distance, or by image within [olo, ohi] (equal steps of 2^shift).
    __device__ __forceinline__ int bin(unsigned o, unsigned ohi, int shift) const {
        if (shift >= 0) return (int)((ohi - o) >> shift);
        const float d = o == top ? 0.0f : f32_from_ord(top) - f32_from_ord(o);
        return min(max((int)(__float_as_uint(d) >> 18) - ((127 - 16) << 5), 0), SBINS - 1);
    }

    // Moves thr up to the last entry of the shortest prefix whose measure reaches `want` (>= 1): MASS: the
    // weight, else the number of entries.  A prefix that never reaches it is left as it is.
    template <bool MASS>
    __device__ void cut(u64 want) {
        unsigned olo = 0, ohi = ~0u;
        int shift = -1;
        u64 base = 0;  // measure of what lies above [olo, ohi]
        for (;;) {
            for (int b = tid; b < SBINS; b += ST) {
                s.n[b] = 0;
                if (MASS) s.lo[b] = s.hi[b] = 0;
            }
            if (tid == 0) s.listed = 0;
            __syncthreads();
            each([&](unsigned o, int i) {
                if (o < olo || o > ohi || key(o, i) < thr) return;
                const int b = bin(o, ohi, shift);
                atomicAdd(&s.n[b], 1u);
                if (MASS) {
                    const u64 w = whole(weight(o));
                    const unsigned l = (unsigned)w, old = atomicAdd(&s.lo[b], l);
                    const unsigned h = (unsigned)(w >> 32) + (old + l < l ? 1u : 0u);
                    if (h) atomicAdd(&s.hi[b], h);
                }
            });
            sync();
            // every CTA adds up its share of the bins and hands the sums to all
            const int share = (SBINS + a.ctas - 1) / a.ctas;
            for (int b = rank * share + tid; b < min((rank + 1) * share, SBINS); b += ST) {
                unsigned n = 0;
                u64 w = 0;
                for (int r = 0; r < a.ctas; ++r) {
                    n += s_get(s_at(&s.n[b], r));
                    if (MASS) w += ((u64)s_get(s_at(&s.hi[b], r)) << 32) + s_get(s_at(&s.lo[b], r));
                }
                for (int r = 0; r < a.ctas; ++r) {
                    s_put(s_at(&s.all_n[b], r), n);
                    if (MASS) s_put(s_at(&s.all_w[b], r), w);
                }
            }
            sync();
            // the bin that reaches the target: thread t holds bin t
            const u64 m = MASS ? s.all_w[tid] : (u64)s.all_n[tid];
            u64 inc = warp_scan(m, lane);
            if (tid == 0) s.found = -1;
            if (lane == 31) s.warp_w[warp] = inc;
            __syncthreads();
            u64 run = base;
            for (int w = 0; w < warp; ++w) run += s.warp_w[w];
            inc += run;
            if (inc >= want && inc - m < want) s.found = tid, s.found_before = inc - m;
            __syncthreads();
            const int b = s.found;
            if (b < 0) return;  // all of it does not reach the target
            base = s.found_before;
            const unsigned n = s.all_n[b];
            if (n <= SLIST) {
                each([&](unsigned o, int i) {
                    const bool in = o >= olo && o <= ohi && key(o, i) >= thr && bin(o, ohi, shift) == b;
                    const unsigned who = __ballot_sync(0xffffffffu, in);
                    if (who == 0) return;
                    unsigned at = 0;
                    if (lane == __ffs(who) - 1) at = s_add(s_at(&s.listed, 0), __popc(who));
                    at = __shfl_sync(0xffffffffu, at, __ffs(who) - 1) + __popc(who & lanemask_lt());
                    if (in) s_put(s_at(&s.list[at], 0), key(o, i));
                });
                sync();
                if (rank == 0) {  // what ranks above mine?  one entry is the last that is needed
                    const u64 k = tid < (int)n ? s.list[tid] : 0ull;
                    if (MASS) {  // the weights beside the keys
                        if (tid < (int)n) s.all_w[tid] = whole(weight(key_ord(k)));
                        __syncthreads();
                    }
                    u64 above = base;
                    for (unsigned e = 0; e < n; ++e)
                        if (s.list[e] > k) above += MASS ? s.all_w[e] : 1ull;
                    if (tid < (int)n && above < want && above + (MASS ? s.all_w[tid] : 1ull) >= want)
                        for (int r = 0; r < a.ctas; ++r) s_put(s_at(&s.cut, r), k);
                }
                sync();
                thr = s.cut;
                return;
            }
            // too many: how far apart are they?
            unsigned least = ~0u, most = 0;
            each([&](unsigned o, int i) {
                if (o >= olo && o <= ohi && key(o, i) >= thr && bin(o, ohi, shift) == b) least = min(least, o), most = max(most, o);
            });
            least = __reduce_min_sync(0xffffffffu, least);
            most = __reduce_max_sync(0xffffffffu, most);
            __syncthreads();
            if (lane == 0) s.warp_n[warp] = least, s.warp_w[warp] = most;
            __syncthreads();
            if (warp == 0) {
                least = __reduce_min_sync(0xffffffffu, s.warp_n[lane]);
                most = __reduce_max_sync(0xffffffffu, (unsigned)s.warp_w[lane]);
                if (lane < a.ctas) {
                    s_put(s_at(&s.slot_a[rank], lane), least);
                    s_put(s_at(&s.slot_b[rank], lane), most);
                }
            }
            sync();
            olo = ~0u, ohi = 0;
            for (int r = 0; r < a.ctas; ++r) olo = min(olo, s.slot_a[r]), ohi = max(ohi, s.slot_b[r]);
            sync();  // the slots may be written again
            if (olo == ohi) {  // equal scores: the first of them, by index
                const u64 each_w = MASS ? whole(weight(olo)) : 1ull;
                const u64 need = (want - base + each_w - 1) / each_w;  // each_w > 0: the bin reaches the target
                if (need < n) {
                    const auto tie = [&](unsigned o, int i) -> u64 { return o == olo && key(o, i) >= thr; };
                    sums(tie);
                    walk(tie, need - 1);
                    if (tid == 0 && s.found >= 0)
                        for (int r = 0; r < a.ctas; ++r) s_put(s_at(&s.cut, r), key(olo, s.found));
                    sync();
                    thr = s.cut;
                } else
                    thr = max(thr, (u64)make_key(olo, ~0u));
                return;
            }
            shift = 0;
            while (((ohi - olo) >> shift) >= SBINS) ++shift;
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(ST) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(s_raw);
    const long long row = blockIdx.x / a.ctas;
    const int rank = blockIdx.x % a.ctas;  // the cluster is the row's CTAs, in order
    Row<T> w = {a, s, reinterpret_cast<T *>(s_raw + sizeof(SampleShared)), static_cast<const T *>(a.logits) + row * a.ld};
    const int tid = w.tid = threadIdx.x, lane = w.lane = tid & 31, warp = w.warp = tid >> 5;
    w.rank = rank;
    w.start = min(rank * a.seg, a.vocab);
    w.len = min(a.seg, a.vocab - w.start);
    w.wlen = ((w.len + SWARPS - 1) / SWARPS + 31) & ~31;

    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float least_in = a.min_p ? a.min_p[row] : 0.0f;
    const float least = fminf(least_in, 1.0f);  // the first is always kept
    const float u = a.u[row];
    const bool bad = !(temp >= 0.0f) || p != p || least_in != least_in || u != u;
    if (temp == 0.0f) temp = 1.0f, k = 1;

    // ---- the row comes in; its largest score ----
    const T *x = w.x + w.start;
    const int held = min(w.len, a.cap);
    unsigned top = 0;
    constexpr int PER = 16 / sizeof(T);
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        const int vecs = held / PER;
        done = vecs * PER;
        constexpr int U = 4;
        for (int v0 = tid; v0 < vecs; v0 += ST * U) {
            uint4 q[U];
#pragma unroll
            for (int e = 0; e < U; ++e)
                if (v0 + e * ST < vecs) q[e] = reinterpret_cast<const uint4 *>(x)[v0 + e * ST];
#pragma unroll
            for (int e = 0; e < U; ++e)
                if (v0 + e * ST < vecs) {
                    reinterpret_cast<uint4 *>(w.data)[v0 + e * ST] = q[e];
                    const T *t = reinterpret_cast<const T *>(&q[e]);
#pragma unroll
                    for (int i = 0; i < PER; ++i) top = max(top, ord_from_f32(Elem<T>::get(t[i])));
                }
        }
    }
    for (int i = done + tid; i < w.len; i += ST) {
        const T t = x[i];
        if (i < held) w.data[i] = t;
        top = max(top, ord_from_f32(Elem<T>::get(t)));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s.warp_n[warp] = top;
    if (a.ctas > 1) w.sync();  // every CTA of the cluster runs before any writes to another
    else __syncthreads();
    if (warp == 0) {
        top = __reduce_max_sync(0xffffffffu, s.warp_n[lane]);
        if (lane < a.ctas) s_put(s_at(&s.slot_a[rank], lane), top);
    }
    w.sync();
    for (int r = 0; r < a.ctas; ++r) top = max(top, s.slot_a[r]);
    if (bad || top <= kNegInf) {  // the whole cluster agrees
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
            if (a.kept) a.kept[row] = 0;
        }
        if (a.ctas > 1) w.sync();
        return;
    }
    w.top = top;
    w.x_top = (double)f32_from_ord(top);
    w.per_t = fmax(1.0 / (double)temp, 1e-300);  // never 0: an infinite distance stays one
    w.thr = make_key(kNegInf + 1, ~0u);
    w.sync();  // the slots may be written again

    // ---- the cuts ----
    if (k > 0 && k < a.vocab) w.template cut<false>((u64)k);
    if (p < 1.0f) {
        const u64 all = w.sums([&](unsigned o, int i) -> u64 { return w.key(o, i) >= w.thr ? w.whole(w.weight(o)) : 0ull; });
        w.sync();
        w.template cut<true>(p <= 0.0f ? 1ull : max((u64)ceil((double)p * (double)all), (u64)1));
    }

    // ---- the draw ----
    u64 count = 0;
    const auto kept_weight = [&](unsigned o, int i) -> u64 {
        if (w.key(o, i) < w.thr) return 0ull;
        const double v = w.weight(o);
        if (least > 0.0f && v < (double)least) return 0ull;
        ++count;
        return w.whole(v);
    };
    const u64 all = w.sums(kept_weight);
    count = warp_sum(count);
    if (lane == 0) s.warp_n[warp] = (unsigned)count;
    const double t = (double)u * (double)all;
    const u64 target = t <= 0.0 ? 0ull : (t >= (double)all ? all - 1 : min((u64)t, all - 1));
    w.walk(kept_weight, target);
    __syncthreads();
    if (s.found >= 0 && tid == 0) {
        a.ids[row] = w.start + s.found;
        if (a.probs) a.probs[row] = (float)((double)s.found_w / (double)all);
    }
    if (a.kept) {
        if (warp == 0) {
            const unsigned n = __reduce_add_sync(0xffffffffu, s.warp_n[lane]);
            if (lane == 0) s_put(s_at(&s.slot_b[rank], 0), n);
        }
        w.sync();
        if (rank == 0 && tid == 0) {
            unsigned n = 0;
            for (int r = 0; r < a.ctas; ++r) n += s.slot_b[r];
            a.kept[row] = (int)n;
        }
    }
}

template <typename T>
static int sample_launch(SampleArgs a, long long rows, int device, cudaStream_t st) {
    constexpr size_t kSmem = 227 * 1024;
    constexpr int kHold = (int)((kSmem - sizeof(SampleShared)) / sizeof(T)) & ~63;
    static bool sized[kMaxDevices];
    static int most[kMaxDevices];  // CTAs of a row
    if (!sized[device]) {
        LK_CUDA(cudaFuncSetAttribute((const void *)k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        LK_CUDA(cudaFuncSetAttribute((const void *)k_sample<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t all = {};  // does a cluster of 16 full CTAs fit on this GPU?
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)(most[device] = SMAX_CTAS);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        all.gridDim = dim3(SMAX_CTAS);
        all.blockDim = dim3(ST);
        all.dynamicSmemBytes = kSmem;
        all.attrs = attr;
        all.numAttrs = 1;
        int fit = 0;
        if (cudaOccupancyMaxActiveClusters(&fit, k_sample<T>, &all) != cudaSuccess || fit < 1) most[device] = 8;  // the portable size
        cudaGetLastError();
        sized[device] = true;
    }
    // as many CTAs to a row as its entries want (4,096 or more each) while the GPU has room for all rows at once, and at
    // least as many as hold the row
    const int sms = sm_count(device);
    a.ctas = 1;
    while (a.ctas < most[device] && (a.vocab > (long long)kHold * a.ctas || (a.vocab >= 8192 * a.ctas && rows * a.ctas * 2 <= sms))) a.ctas *= 2;
    a.seg = (int)round_up((a.vocab + a.ctas - 1) / a.ctas, 64);
    a.cap = std::min(a.seg, kHold);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * a.ctas));
    cfg.blockDim = dim3(ST);
    cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)a.cap * sizeof(T);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launch_cfg("lk_sample", k_sample<T>, cfg, a);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_sample(int device, int dtype, int64_t rows, int64_t vocab, const void *d_logits, int64_t ld,
                         const float *d_temperature, const int32_t *d_top_k, const float *d_top_p, const float *d_min_p,
                         const float *d_u, int64_t *d_ids, float *d_probs, int32_t *d_kept, void *stream) {
    if (!float_type(dtype)) return fail(LK_EINVAL, "lk_sample: dtype is LK_F32, LK_F16 or LK_BF16");
    if (rows < 0 || vocab < 0) return fail(LK_EINVAL, "lk_sample: bad size");
    if (vocab > LK_SAMPLE_MAX_VOCAB) return fail(LK_ERANGE, "lk_sample: vocab is limited to LK_SAMPLE_MAX_VOCAB (16777216)");
    if (rows > 0x7ffffff) return fail(LK_ERANGE, "lk_sample: more than 2^27-1 rows");
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
    SampleArgs a = {d_logits, ld, (int)vocab, 1, 0, 0, d_temperature, d_top_p, d_min_p, d_u, d_top_k,
                    reinterpret_cast<long long *>(d_ids), d_probs, d_kept, (double)(1ull << (63 - bits))};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == LK_F32) return sample_launch<float>(a, rows, device, st);
    if (dtype == LK_F16) return sample_launch<__half>(a, rows, device, st);
    return sample_launch<__nv_bfloat16>(a, rows, device, st);
}
