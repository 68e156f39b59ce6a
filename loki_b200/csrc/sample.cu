// One draw per row of scores: temperature, top-k, top-p, min-p, from given random numbers.
//
// Every filter keeps a prefix of the row's order (score descending, index ascending), so what is kept is
// described by its last entry: a 64-bit ranking key (score image, ~index) at or above which entries are kept.
// Weights w = exp((x - max) / T) are computed in float64 and summed as 64-bit integers, w * 2^F with sums below
// 2^62 and F <= 49: sums do not depend on their order (shared-memory atomics, warps, CTAs), and the prefix
// that a cut finds and the running sum that a draw walks agree to the last bit.  Each weight is rounded by 2^-(F+1) of the
// largest at most, and by 2e-12 of itself (the series), so that a sum over n entries is off by n 2^-(F+1) at most, all in one direction
// where their scores are equal.  Up to 2^18 entries F follows from their number, n 2^F <= 2^62: 2^-27 of the largest weight.
// A longer row takes F from a bound on its own sum, the largest weight that each thread has seen times its entries: where F is 49
// the sums of 2^24 entries are off by 2^-26 of the largest weight, elsewhere by 2^-28 of the sum, as the bound is at most 1,040 times that.
// 2^-26 of the row's weight is a quarter of the step between two neighbouring values of u below 1.
//
// A cluster of CTAs owns a row.  Each loads one stretch of it into its shared memory (what does not fit is read
// again from L2), so scores cross HBM once; every later pass runs over shared memory, and the CTAs
// exchange maxima, histograms and sums through distributed shared memory.  Bound: instructions per entry
// and pass, so passes are what is saved:
//
// * Few candidates.  With a top-k, the k-th largest of the threads' maxima bounds the k-th score from below: one
//   pass gathers what reaches that bound in one CTA, and if that is 1,024 entries or fewer they are sorted there and
//   all filters and the draw are settled among them.  Without a top-k the same happens when the bins that
//   hold top_p of the weight have that few entries.
// * Many.  A cut by count or weight: entries fall into 1,024 bins by the distance d = (max - x) / T, 128 bins to a
//   factor of two from 1/8 to 32 (the bits of d without the low ones: monotone in x, and fine where a softmax
//   has its weight; few entries of a warp meet in one bin).  The bin in which the measure reaches its target is
//   cut again by the next bits of d, then by the bits of x, until at most 1,024 entries are left to be sorted, or all
//   are equal and are cut by index.  A cut by weight first tries to do with one pass over the weights (look()).
//   Then a pass sums the kept weights by warp and CTA, if that look has not, and the draw walks down those sums.
//
// Measured, 64 x 131,072 bf16 scores, rows cut by top-p 0.9 alone, of 56 us: loading 3, the maximum 2.5, counting into bins 9, the
// pass over the weights with what is joined after it 21.5, gathering 5.5, sorting 5, the walk 2.5; the rest are meetings.
#include <cfloat>
#include <type_traits>

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
    int unit_bits;  // F, or what it is at least
};

constexpr unsigned kNegInf = 0x007fffffu;  // image of -infinity; NaN (0) is below it
constexpr int ST = 1024, SWARPS = ST / 32;
constexpr int SBINS = 1024;                // one thread per bin
constexpr int SLIST = 1024;                // one thread per candidate
constexpr int SMAX_CTAS = 16;
constexpr int kWide = 1 << 18;             // rows longer than this choose F by their scores (WIDE)
constexpr unsigned kSlack = 256;           // look(): entries to either side of an estimate
constexpr int SD_SHIFT = 16, SD_BASE = (127 - 3) << 7;  // bins by d: exponent and 7 bits, from 2^-3 to 2^5
using u64 = unsigned long long;
// Measured with a top-p alone, 1 to 512 rows of 4,096 to 1,000,000 scores: a CTA's time per entry over all passes, and for one that
// its shared memory does not hold, its start and its sorts, and what the meetings of a cluster add, and of one of more
// than eight.  A row with a small top-k costs less per entry, but the host does not see the filters.  Over 92 shapes and filters the
// number of CTAs that follows costs 1.3 % against the best uniform number on average, 25 % at worst (100 rows of 151,936, mixed filters).
constexpr double SAMPLE_ENTRY_NS = 0.5, SAMPLE_AWAY_NS = 0.15, SAMPLE_CTA_NS = 15000.0, SAMPLE_MEET_NS = 8000.0, SAMPLE_WIDE_NS = 6000.0;

struct alignas(16) SampleShared {
    unsigned lo[SBINS], hi[SBINS], n[SBINS];   // this CTA's bins: weights (two words), entries
    u64 all_w[SBINS];                          // the row's bins
    unsigned all_n[SBINS];
    u64 list[SLIST];                           // this CTA's candidates
    u64 sorted[SLIST];                         // scratch of the sort
    double octave[128][8];                     // 2^(F + j/128), eight times
    u64 warp_w[SWARPS];
    unsigned warp_n[SWARPS];
    u64 above_w[SWARPS];                       // look(): what lies above the cut's place, by warp
    unsigned above_n[SWARPS];
    u64 slot_w[SMAX_CTAS], slot_v[SMAX_CTAS];  // one word from every CTA of the row
    unsigned slot_top[SMAX_CTAS], slot_n[SMAX_CTAS], slot_a[SMAX_CTAS], slot_b[SMAX_CTAS];
    unsigned noted;
    unsigned n_before, n_upto, n_next;         // look(): entries above a bin, down to its end and to the next one's
    int first, last;
    u64 cut;                                   // a decision of the first CTA, or of the one that holds an entry
    u64 found_w, found_before, floor;
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
__device__ __forceinline__ u64 s_get64(unsigned at) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
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

// One step of a bitonic sort of one key per lane: this lane's stretch of 2 * STRIDE keys keeps the larger keys low (or high).
template <int STRIDE>
__device__ __forceinline__ void lane_step(u64 &k, bool down) {
    const u64 o = shfl_xor_u64(k, STRIDE);
    if ((k < o) == (((threadIdx.x & STRIDE) == 0) == down)) k = o;
}
// Keys sorted, largest first, one per thread (0 = none; n of them, in the first threads); every thread of the CTA takes part.
// Strides below 32 by shuffles, wider ones through shared memory.
__device__ __noinline__ u64 block_sort(SampleShared &s, u64 k, int n) {
    const int tid = threadIdx.x;
    int size_max = 32;
    while (size_max < n) size_max <<= 1;
    const bool used = tid < size_max;  // whole warps
    if (used) {
        lane_step<1>(k, (tid & 2) == 0);
        lane_step<2>(k, (tid & 4) == 0), lane_step<1>(k, (tid & 4) == 0);
        lane_step<4>(k, (tid & 8) == 0), lane_step<2>(k, (tid & 8) == 0), lane_step<1>(k, (tid & 8) == 0);
        lane_step<8>(k, (tid & 16) == 0), lane_step<4>(k, (tid & 16) == 0), lane_step<2>(k, (tid & 16) == 0), lane_step<1>(k, (tid & 16) == 0);
    }
    for (int size = 32; size <= size_max; size <<= 1) {
        const bool down = (tid & size) == 0;  // this stretch descends
        for (int stride = size >> 1; stride >= 32; stride >>= 1) {
            __syncthreads();
            if (used) s.sorted[tid] = k;
            __syncthreads();
            if (used) {
                const u64 o = s.sorted[tid ^ stride];
                if ((k < o) == (((tid & stride) == 0) == down)) k = o;
            }
        }
        if (used) lane_step<16>(k, down), lane_step<8>(k, down), lane_step<4>(k, down), lane_step<2>(k, down), lane_step<1>(k, down);
    }
    return k;
}
// Inclusive running sum over the threads of the CTA.
__device__ __noinline__ u64 block_scan(SampleShared &s, u64 v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) s.warp_w[warp] = v;
    __syncthreads();
    const u64 other = warp_scan(s.warp_w[lane], lane);
    return warp == 0 ? v : v + __shfl_sync(0xffffffffu, other, warp - 1);
}

// One row, as the CTAs of its cluster see it.
template <typename T, bool WIDE>
struct Row {
    static constexpr int PER = 16 / sizeof(T);  // entries of a 16-byte group
    const SampleArgs &a;
    SampleShared &s;
    T *data;        // this CTA's stretch in shared memory, `cap` entries of it, padded with NaN to a whole group
    const T *x;     // this CTA's stretch in global memory
    int rank, start, len, wlen, tid, lane, warp;
    float top;      // the largest score
    float bottom;   // a score so far below it that it weighs nothing
    bool alone;     // nothing else weighs: it is +infinity, or T is that small
    double top_wide;
    double octaves; // 128 / (T ln 2): a score in 128ths of an octave
    double whole;   // 1.5 * 2^52 - N: adding it rounds to a whole number in the low word
    float temp, per_t;  // T, 1 / T
    int unit_bits;      // F
    float split;        // look() has summed the weights of what is above this by warp
    bool summed;        // those sums have become the ones of all that is kept
    u64 floor;      // min_p: the lowest key that it keeps
    u64 thr;        // entries with a key at or above this are kept
    float thr_x;    // its score and its index
    int thr_i;

    __device__ __forceinline__ void sync() const {
        if (a.ctas > 1) {
            asm volatile("barrier.cluster.arrive;" ::: "memory");
            asm volatile("barrier.cluster.wait;" ::: "memory");
        } else
            __syncthreads();
    }
    __device__ __forceinline__ u64 key(float v, int i) const { return make_key(ord_from_f32(v), (unsigned)(start + i)); }
    __device__ __forceinline__ void keep_from(u64 k) {
        thr = k;
        thr_x = f32_from_ord(key_ord(k));
        thr_i = (int)min((long long)key_slot(k) - start, 0x7fffffffll);  // as a local index
    }
    // NaN compares false; -infinity is below every threshold
    __device__ __forceinline__ bool kept(float v, int i) const { return v > thr_x || (v == thr_x && i <= thr_i); }
    __device__ __forceinline__ void kept4(const float (&v)[4], int i, bool (&k)[4]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = v[e] >= thr_x;
        if (thr_i != 0x7fffffff) {  // a cut among equals
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = k[e] && !(v[e] == thr_x && i + e > thr_i);
        }
    }
    __device__ __forceinline__ float entry(int i) const { return Elem<T>::get(i < a.cap ? data[i] : x[i]); }

    // About exp((v - than) / T), for v <= than.
    __device__ __forceinline__ float lighter(float v, float than) const {
        return v == than ? 1.0f : than == CUDART_INF_F ? 0.0f : exp2f((float)(((double)v - (double)than) * octaves / 128.0));
    }
    // w * 2^F of a score, rounded, where others than the largest weigh.  Tang's scheme (ACM TOMS 15, 1989): with y = x / T / ln 2 *
    // 128 = N + n + r, n whole, |r| <= 1/2, N the whole number next to the largest y:  w = 2^(n div 128) * 2^((n mod 128) / 128) *
    // e^(r ln 2 / 128), the middle factor from a table, the last by its series to the third power (next term 2e-12 at most).
    // All weights of a row share a factor within 2^(1/256) of 1 (the largest y is not whole), which no quotient of weights
    // sees.  Roundings to whole numbers are done by adding constants, powers of two on the bits.
    // Bound: issue slots, like the passes that call it (about 8 of the 20 us of a pass over 65,536 scores).  The table has eight
    // copies, so that the lanes of a warp seldom meet in a bank (with one copy of 1,024 entries the banks took 17 clocks a warp).
    // plus() returns 2^52 + w * 2^F, a whole number below 2^53.
    static constexpr double kOne = 4503599627370496.0;  // 2^52
    __device__ __forceinline__ double plus(float v) const {
        const double x = (double)fmaxf(v, bottom);
        const double t = fma(x, octaves, whole);
        const double r = fma(x, octaves, whole - t);
        const int n = __double2loint(t);
        constexpr double c = 0.693147180559945309417232 / 128;
        const double q = fma(r, fma(r, fma(r, c * c * c / 6, c * c / 2), c), 1.0);
        const double f = s.octave[n & 127][lane & 7];
        const double scaled = __hiloint2double(__double2hiint(f) + (int)(((unsigned)n & ~127u) << 13), __double2loint(f));
        return fma(q, scaled, kOne);
    }
    static __device__ __forceinline__ u64 whole_of(double p) { return (u64)__double_as_longlong(p) - 0x4330000000000000ull; }
    __device__ __forceinline__ u64 weight(float v) const { return whole_of(plus(v)); }
    // The same for any row.
    __device__ __forceinline__ u64 weight_of(float v) const {
        if (alone) return v == top ? 1ull << unit_bits : 0ull;
        return weight(v);
    }
    // Of four scores; those that are not kept weigh nothing.
    __device__ __forceinline__ void weights(const float (&v)[4], const bool (&k)[4], u64 (&w)[4]) const {
        if (alone) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = k[e] && v[e] == top ? 1ull << unit_bits : 0ull;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 m = weight(v[e]);
                w[e] = k[e] ? m : 0ull;
            }
        }
    }

    // f(four scores, local index of the first) for the entries of this warp's stretch, NaN for those past its end.  Four
    // at a time, because their weights are then computed side by side; one copy of f in the code, because a kernel this
    // short waits for its instructions.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int lo = warp * wlen, hi = min(lo + wlen, len);
        const bool groups = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
        using Group = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
        const auto fetch = [&](int i) {
            Group q;
            if (i < a.cap) return *reinterpret_cast<const Group *>(data + i);  // whole: the stretch is padded with NaN
            if (groups && i + 4 <= hi) return *reinterpret_cast<const Group *>(x + i);
            T *t = reinterpret_cast<T *>(&q);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = i + e < hi ? x[i + e] : Elem<T>::put(CUDART_NAN_F);
            return q;
        };
        int i = lo + lane * 4;
        Group next = {};
        if (i < hi) next = fetch(i);
#pragma unroll 1
        for (; i < hi; i += 128) {
            const Group q = next;
            if (i + 128 < hi) next = fetch(i + 128);  // under way while this one is worked on
            const T *t = reinterpret_cast<const T *>(&q);
            const float v[4] = {Elem<T>::get(t[0]), Elem<T>::get(t[1]), Elem<T>::get(t[2]), Elem<T>::get(t[3])};
            f(v, i);
        }
    }

    // A thread's sum of weights.  It can be taken in float64 without rounding (one instruction instead of two, and in a pipe with room)
    // where it stays below 2^53: of n entries a thread has n / 1,024 and 5 at most, F + log2 n <= 62 and F <= 49.  A WIDE row's F says
    // nothing about a thread's share: there four weights, below 2^52, are added in float64 and then to a whole number.
    struct Sum {
        double part = WIDE ? kOne : 0.0;
        u64 before = 0;
        __device__ __forceinline__ void add(double w) { part += w; }
        __device__ __forceinline__ void next() {  // behind four weights at most
            if constexpr (WIDE) before += whole_of(part), part = kOne;
        }
        __device__ __forceinline__ u64 get() const { return WIDE ? before : (u64)part; }
    };

    // Sum over the entries that keep(scores, index, out) says of their weights (MASS) or their number; warp_w keeps this CTA's warps'
    // sums and slot_w the CTAs'.  *mine: how many of this thread's entries there are.
    template <bool MASS, typename K>
    __device__ __forceinline__ u64 sums(K keep, unsigned *mine) const {
        Sum sum;
        unsigned n = 0;
        const double one = (double)(1ull << unit_bits);
        each([&](const float (&v)[4], int i) {
            bool k[4];
            keep(v, i, k);
            if (!(k[0] | k[1] | k[2] | k[3])) return;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k[e]) ++n;
            if (!MASS) return;
            if (alone) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k[e] && v[e] == top) sum.add(one);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double w = plus(v[e]) - kOne;
                    if (k[e]) sum.add(w);
                }
            }
            sum.next();
        });
        *mine = n;
        u64 w = MASS ? sum.get() : (u64)n;
        if (MASS && split < CUDART_INF_F && lane == 0) w += s.above_w[warp], *mine += s.above_n[warp];
        return join_sums(warp_sum(w));
    }
    // From the warps' sums: warp_w, slot_w, and the sum over the row.
    __device__ __forceinline__ u64 join_sums(u64 w) const {
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
    // The entry at which the running sum (in the order of the indexes) first exceeds `target`, which is below the sum
    // that sums() has just returned for the same entries: the CTA that holds it sets found (local index) and found_w (its
    // measure); in the others found is -1.  No meeting of the cluster.
    template <bool MASS, typename K>
    __device__ __forceinline__ void walk(K keep, u64 target) const {
        const auto f = [&](float v, int i) -> u64 { return keep(v, i) ? (MASS ? weight_of(v) : 1ull) : 0ull; };
        __syncthreads();
        if (tid == 0) s.found = -1;
        u64 before = 0;
        for (int r = 0; r < rank; ++r) before += s.slot_w[r];
        const bool mine = before <= target && target < before + s.slot_w[rank];
        __syncthreads();
        if (!mine) return;
        int lo = 0, n = wlen;  // first the stretch of a warp, then a 32nd of that, then its entries
        for (int level = 0;; ++level) {
            const u64 w_at = s.warp_w[lane], inc_at = warp_scan(w_at, lane) + before;
            const unsigned past = __ballot_sync(0xffffffffu, inc_at > target);
            const int at = past ? __ffs(past) - 1 : 31;  // there is one
            before = shfl_u64(inc_at - w_at, at);
            lo += at * n;
            if (level == 1) break;
            const int end = min(lo + n, len);
            n = ((n + SWARPS - 1) / SWARPS + 31) & ~31;
            u64 w = 0;
            for (int i0 = lo + warp * n; i0 < min(lo + (warp + 1) * n, end); i0 += 32) {
                const int i = i0 + lane;
                if (i < end) w += f(entry(i), i);
            }
            w = warp_sum(w);
            __syncthreads();
            if (lane == 0) s.warp_w[warp] = w;
            __syncthreads();
        }
        if (warp == 0) {
            for (int i0 = lo; i0 < min(lo + n, len); i0 += 32) {
                const int i = i0 + lane;
                const u64 w = i < len ? f(entry(i), i) : 0ull;
                const u64 inc = warp_scan(w, lane) + before;
                const unsigned past = __ballot_sync(0xffffffffu, inc > target);
                if (past) {
                    if (lane == __ffs(past) - 1) s.found = i, s.found_w = w;
                    break;
                }
                before = __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        __syncthreads();
    }

    // The lists hold every entry that may be kept (n of them): in the first CTA, all filters and the draw.  `all`: the weight
    // that top_p refers to, 0 = that of the k first.
    __device__ void finish(long long row, int n, int k, float p, float u, u64 all) const {
        const u64 mine = block_sort(s, fetch(), n);  // thread t holds the entry of rank t
        const float v = f32_from_ord(key_ord(mine));
        const bool in = tid < n && (k <= 0 || tid < k);
        const u64 w = in ? weight_of(v) : 0ull;
        const u64 inc = block_scan(s, w);
        if (tid == ST - 1) s.found_before = inc;
        __syncthreads();
        if (all == 0) all = s.found_before;
        const u64 want = p < 1.0f ? prefix(p, all) : ~0ull;
        const bool keep = in && inc - w < want && (tid == 0 || mine >= floor);
        const int count = __syncthreads_count(keep);
        if (tid == count - 1) s.found_w = inc;
        s.all_w[tid] = w;
        const unsigned slot = key_slot(mine);
        // the kept ones by index: largest first of ~(index, rank)
        const u64 by_index = block_sort(s, keep ? ~(((u64)slot << 10) | (unsigned)tid) : 0ull, count);
        __syncthreads();
        const u64 total = s.found_w;
        const unsigned from = (unsigned)~by_index & 1023u;
        const u64 w2 = tid < count ? s.all_w[from] : 0ull;
        const u64 run = block_scan(s, w2);
        const u64 target = aim(u, total);
        if (run - w2 <= target && target < run) {
            a.ids[row] = (long long)((~by_index) >> 10);
            if (a.probs) a.probs[row] = (float)((double)w2 / (double)total);
            if (a.kept) a.kept[row] = count;
        }
    }
    // The lowest key with w >= min_p, i.e. (x - max) / T >= log(min_p): a warp tries 32 images at a time.
    __device__ __forceinline__ u64 lowest(float min_p) const {
        const double end = log((double)min_p);
        unsigned lo = kNegInf + 1, hi = ord_from_f32(top);  // the largest score is always kept
        while (lo < hi) {
            const unsigned step = (hi - lo) / 32 + 1, mid = lo + min(lane * step, hi - lo);
            const bool in = mid == hi || ((double)f32_from_ord(mid) - top_wide) * (octaves * (0.693147180559945309417232 / 128)) >= end;
            const int first = __ffs(__ballot_sync(0xffffffffu, in)) - 1;  // lanes ascend: the first that is kept, if any
            if (first < 0) lo += 31 * step + 1;
            else {
                hi = __shfl_sync(0xffffffffu, mid, first);
                if (first > 0) lo = __shfl_sync(0xffffffffu, mid, first - 1) + 1;
                else break;  // lo itself
            }
        }
        return make_key(hi, ~0u);
    }
    // Shares of a sum, without a rounding on the way: where weights are equal a share can be met exactly, and float64 would round a sum past 2^53 to
    // one side or the other.

    // The least weight that a prefix with the share p of `all` has: p * all rounded up, in whole numbers.
    static __device__ __forceinline__ u64 prefix(float p, u64 all) {
        if (p <= 0.0f) return 1ull;
        const unsigned bits = __float_as_uint(p), e = max(bits >> 23, 1u);
        const u64 m = bits < 0x800000u ? bits : (bits & 0x7fffffu) | 0x800000u;  // p = m * 2^-s
        const int s = 150 - (int)e;                                              // 24 at least: p is below 1
        const u64 lo = all * m, hi = __umul64hi(all, m);                         // hi is below 2^24
        if (s < 64) return (hi << (64 - s) | lo >> s) + ((lo & ((1ull << s) - 1)) != 0 ? 1 : 0);
        const u64 whole = s < 128 ? hi >> (s - 64) : 0ull;
        return whole + (lo != 0 || (s < 128 ? whole << (s - 64) != hi : hi != 0) ? 1 : 0);  // p * all > 0: 1 at least
    }
    // u * total rounded down, which the running sum of the entry drawn exceeds: in float64 with what its product loses.  (In whole numbers, or with the
    // first test on u alone, the compiler schedules the loop of sums() before it worse: 4 x 16,000,000 bfloat16 scores 322 us instead of 282.)
    static __device__ __forceinline__ u64 aim(float u, u64 total) {
        if ((double)u * (double)total <= 0.0) return 0ull;
        const double v = (double)fminf(u, 1.0f), low = (double)(unsigned)(total & 1023ull), most = (double)(total & ~1023ull);  // exact: below 2^62
        const double h = v * most, whole = ::floor(h), rest = (h - whole) + (fma(v, most, -h) + v * low);
        return min((u64)whole + (u64)(long long)::floor(rest), total - 1);
    }

    // Every CTA adds up its share of the row's bins and hands the sums to all: thread (bin, CTA r) reads that bin of r's
    // and, after the 2^g >= ctas threads of a bin have added up, writes the sum to r.
    template <bool MASS>
    __device__ __forceinline__ void join_bins() const {
        if (a.ctas == 1) {
            __syncthreads();
            s.all_n[tid] = s.n[tid];
            if (MASS) s.all_w[tid] = ((u64)s.hi[tid] << 32) + s.lo[tid];
            __syncthreads();
            return;
        }
        sync();
        int wide = 2;
        while (wide < a.ctas) wide <<= 1;
        const int r = tid & (wide - 1), share = (SBINS + a.ctas - 1) / a.ctas, end = min((rank + 1) * share, SBINS);
        for (int b0 = rank * share; b0 < end; b0 += ST / wide) {
            const int b = b0 + tid / wide;
            const bool there = b < end && r < a.ctas;
            unsigned n = 0;
            u64 w = 0;
            if (there) {
                n = s_get(s_at(&s.n[b], r));
                if (MASS) w = ((u64)s_get(s_at(&s.hi[b], r)) << 32) + s_get(s_at(&s.lo[b], r));
            }
            for (int d = 1; d < wide; d <<= 1) {
                n += __shfl_xor_sync(0xffffffffu, n, d);
                if (MASS) w += shfl_xor_u64(w, d);
            }
            if (there) {
                s_put(s_at(&s.all_n[b], r), n);
                if (MASS) s_put(s_at(&s.all_w[b], r), w);
            }
        }
        sync();
    }
    template <bool MASS>
    __device__ __forceinline__ void clear_bins() const {
        s.n[tid] = 0;
        if (MASS) s.lo[tid] = s.hi[tid] = 0;
        if (tid == 0) s.noted = 0;
        __syncthreads();
    }
    // The bin in which the running measure (from `base` on) reaches `want`, -1 if none; found_before = what lies above it.
    __device__ __forceinline__ int reach(u64 m, u64 base, u64 want) const {
        if (tid == 0) s.found = -1;
        const u64 inc = block_scan(s, m) + base;
        if (inc >= want && inc - m < want) s.found = tid, s.found_before = inc - m;
        __syncthreads();
        return s.found;
    }
    __device__ __forceinline__ unsigned distance(float v) const { return __float_as_uint(v == top ? 0.0f : (top - v) * per_t); }
    static __device__ __forceinline__ int first_bin(unsigned d) { return min(max((int)(d >> SD_SHIFT) - SD_BASE, 0), SBINS - 1); }

    // The candidates of bin b and above, in the lists: d below an end.  Their number (which may be more than fit).
    __device__ __forceinline__ unsigned gather_to(int b) const {
        const unsigned end = (unsigned)(SD_BASE + b + 1) << SD_SHIFT;
        const float before = b >= SBINS - 1 ? CUDART_INF_F : __uint_as_float(end);
        // a score below all candidates, for a quick look: the end of the bins with room for the roundings
        const double reach_d = (double)before * (double)temp;
        float near = (float)(top_wide - reach_d - 1e-5 * (reach_d + fabs(top_wide)) - 1e-37);
        if (!(near < CUDART_INF_F)) near = -CUDART_INF_F;
        each([&](const float (&v)[4], int i) {
            if (!(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= near)) return;  // fmaxf passes over NaN
            bool in[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) in[e] = (top - v[e]) * per_t < before || v[e] == top;  // false for NaN and -infinity
            note(in, v, i);
        });
        return deliver();
    }
    // Candidates go to this CTA's own list; deliver() tells all CTAs how many there are (more than SLIST: some are missing),
    // and the first CTA fetches the lists: thread t has candidate t.
    __device__ __forceinline__ void note(const bool (&in)[4], const float (&v)[4], int i) const {
        if (!(in[0] | in[1] | in[2] | in[3])) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (in[e]) {
                const unsigned at = atomicAdd(&s.noted, 1u);
                if (at < SLIST) s.list[at] = key(v[e], i + e);
            }
    }
    __device__ __forceinline__ unsigned deliver() const {
        __syncthreads();
        if (tid < a.ctas) s_put(s_at(&s.slot_n[rank], tid), s.noted);
        sync();
        unsigned n = 0;
        for (int r = 0; r < a.ctas; ++r) n += s.slot_n[r];
        return n;
    }
    __device__ __forceinline__ u64 fetch() const {
        unsigned at = tid;
        for (int r = 0; r < a.ctas; ++r) {
            if (at < s.slot_n[r]) return s_get64(s_at(&s.list[at], r));
            at -= s.slot_n[r];
        }
        return 0ull;
    }

    // The first look of a cut by weight, at the price of one pass over the weights: the entries of each bin are counted, which
    // with the mean weight of a bin says to a thousandth where the cut is, and then one pass sums the kept weights of all, of what
    // lies above a stretch of scores around that place (by warp, for the draw; `split` is the stretch's upper end), and bins that
    // stretch finely by the scores' images.  The sums are exact: they show whether the cut is in there (1: found, found_before
    // and all_n, all_w of the fine bins of 2^sub images from ohi down are set), else the cut is made from the beginning (0).
    // 2: there are at most SLIST entries down to there, and they are in the lists.  3: min_p cuts higher, and all that it keeps has
    // been summed by warp.
    __device__ __forceinline__ int look(float p, bool whole_row, u64 *all, u64 *want, unsigned *olo, unsigned *ohi, int *sub, int *listed) {
        clear_bins<false>();
        each([&](const float (&v)[4], int i) {
            bool k[4];
            kept4(v, i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k[e]) atomicAdd(&s.n[first_bin(__float_as_uint((top - v[e]) * per_t))], 1u);  // distance(), as top is finite
        });
        join_bins<false>();
        const auto edge = [](int b) { return __uint_as_float((unsigned)(SD_BASE + b) << SD_SHIFT); };
        const float lo = tid == 0 ? 0.0f : edge(tid), hi = edge(tid + 1);
        const float mean = (__expf(-lo) - __expf(-hi)) / (hi - lo);
        const u64 m = __float2ull_rn((float)s.all_n[tid] * mean * 1073741824.0f);
        const u64 inc = block_scan(s, m);
        if (tid == ST - 1) s.cut = inc;
        __syncthreads();
        const u64 near = max((u64)((double)fmaxf(p, 0.0f) * (double)s.cut), (u64)1);
        const int b = reach(m, 0ull, near);
        if (b < 0 || b >= SBINS - 2) return 0;
        // The estimate is off where few entries carry the weight, so the stretch goes on from the place's bin until it has kSlack
        // more entries, down through bin `last` and up through bin `first` (0 or -1: from the largest score on).  When all that
        // may be kept can be listed, the list ends with the last bin that keeps it to an eighth more than what the estimate says.
        const unsigned n = s.all_n[tid], upto = (unsigned)block_scan(s, n), above_n = upto - n;
        if (tid == 0) s.first = -1, s.last = SBINS - 2;
        if (tid == b) s.n_before = above_n, s.n_upto = upto;
        if (tid == b + 1) s.n_next = upto;
        __syncthreads();
        const bool few = whole_row && s.n_next <= SLIST;
        const unsigned down = few ? min(s.n_next + s.n_next / 8 + 32, (unsigned)SLIST) : s.n_upto + kSlack - 1;
        if (upto > down && above_n <= down && tid <= SBINS - 2) s.last = few ? tid - 1 : tid;
        if (s.n_before >= kSlack && above_n <= s.n_before - kSlack && upto > s.n_before - kSlack) s.first = tid;
        __syncthreads();
        const int first = s.first, last = s.last;
        // the ends of the stretch; how they are rounded does not matter
        const float d0 = b == 0 ? 0.0f : edge(b), d1 = edge(b + 1);
        const float in_bin = (float)s.all_n[b] * ((__expf(-d0) - __expf(-d1)) / (d1 - d0)) * 1073741824.0f;
        const float part = fminf(fmaxf((float)(near - s.found_before) / in_bin, 0.0f), 1.0f);
        const float place = d0 + part * (d1 - d0), side = edge(b + 2) - edge(b + 1);
        const bool dense = s.all_n[b] >= 2 * kSlack;
        const float above_d = dense && first == b - 1 ? place - side : edge(max(first, 0));
        const float below_d = dense && last == b + 1 ? place + side : edge(last + 1);
        const float above_x = few || first <= 0 ? CUDART_INF_F : (float)(top_wide - (double)above_d * (double)temp);
        // (a list must not take in a value on the bin's edge, of which there may be hundreds)
        const double below_wide = top_wide - (double)below_d * (few ? 1.0 - 1e-6 : 1.0) * (double)temp;
        // min_p cuts higher than that: it is enough that what it keeps weighs less than the target
        const bool by_floor = !few && floor > thr && f32_from_ord(key_ord(floor)) > above_x;
        const float below_x = by_floor ? CUDART_INF_F : fmaxf(few ? __double2float_ru(below_wide) : (float)below_wide, -FLT_MAX);
        *ohi = ord_from_f32(fminf(above_x, top));
        *olo = ord_from_f32(below_x);
        *sub = 0;
        while (((*ohi - *olo) >> *sub) >= SBINS) ++*sub;
        __syncthreads();
        clear_bins<true>();
        Sum sum_all, sum_above;
        unsigned n_above = 0;
        const float upper = few ? nextafterf(below_x, -CUDART_INF_F) : by_floor ? nextafterf(f32_from_ord(key_ord(floor)), -CUDART_INF_F) : above_x;
        each([&](const float (&v)[4], int i) {
            bool k[4], in[4];
            double w[4];
            kept4(v, i, k);
            if (!(k[0] | k[1] | k[2] | k[3])) return;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = plus(v[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double whole = w[e] - kOne;
                const bool over = k[e] && v[e] > upper;
                if (k[e]) sum_all.add(whole);
                if (over) sum_above.add(whole), ++n_above;
                in[e] = few ? over : k[e] && !over && v[e] >= below_x;
            }
            sum_all.next(), sum_above.next();
            if (few) note(in, v, i);
            else if (in[0] | in[1] | in[2] | in[3]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (in[e]) {
                        const int at = (int)((*ohi - ord_from_f32(v[e])) >> *sub);
                        atomicAdd(&s.n[at], 1u);
                        const u64 m = whole_of(w[e]);
                        const unsigned l = (unsigned)m, old = atomicAdd(&s.lo[at], l);
                        const unsigned h = (unsigned)(m >> 32) + (old + l < l ? 1u : 0u);
                        if (h) atomicAdd(&s.hi[at], h);
                    }
            }
        });
        u64 w_all = warp_sum(sum_all.get()), w_above = warp_sum(sum_above.get());
        n_above = __reduce_add_sync(0xffffffffu, n_above);
        if (lane == 0) s.warp_w[warp] = w_all, s.above_w[warp] = w_above, s.above_n[warp] = n_above;
        __syncthreads();
        if (warp == 0) {
            w_all = warp_sum(s.warp_w[lane]);
            w_above = warp_sum(s.above_w[lane]);
            if (lane < a.ctas) {
                s_put(s_at(&s.slot_w[rank], lane), w_all);
                s_put(s_at(&s.slot_v[rank], lane), w_above);
            }
        }
        if (few) *listed = (int)deliver();
        else if (by_floor) sync();
        else join_bins<true>();
        u64 above = 0;
        *all = 0;
        for (int r = 0; r < a.ctas; ++r) *all += s.slot_w[r], above += s.slot_v[r];
        *want = prefix(p, *all);
        sync();  // the slots may be written again
        if (few) return above >= *want && *listed <= SLIST ? 2 : 0;
        if (by_floor) return above < *want ? 3 : 0;
        if (above >= *want || reach(s.all_w[tid], above, *want) < 0) return 0;
        split = above_x;
        return 1;
    }

    // MASS: moves thr up to the last entry of the shortest prefix that holds the share p of the kept weight.
    // Else: to the k-th entry.  Returns the number of candidates when all that may be kept is in the
    // lists instead (`whole`: thr is still at the row's end), with the row's weight in *all; 0 when thr has been moved.
    template <bool MASS>
    __device__ int cut(int k, float p, bool whole, u64 *all) {
        u64 want = (u64)k, base = 0;  // base: measure of what lies above the current bin
        // the entries looked at: d >> in == pre (by distance), or image in [olo, ohi]; their bins: (d >> sub) - from
        int in = 31, sub = SD_SHIFT;
        unsigned pre = 0, from = SD_BASE, olo = 0, ohi = 0;
        bool by_image = false, looked = false;
        int seen = 0;
        if (MASS && !alone) {
            int listed;
            seen = look(p, whole, all, &want, &olo, &ohi, &sub, &listed);
            if (seen == 2) return listed;
            if (seen == 3) {
                keep_from(floor);
                summed = true;
                return 0;
            }
            if (seen == 1) looked = by_image = true;
            else sub = SD_SHIFT;
        }
        for (int level = looked ? 1 : 0;; ++level) {
            if (!looked) clear_bins<MASS>();
            const auto bin = [&](float v) -> int {  // -1: not among those looked at
                if (by_image) {
                    const unsigned o = ohi - ord_from_f32(v);
                    return o <= ohi - olo ? (int)(o >> sub) : -1;
                }
                const unsigned d = distance(v);
                const int b = (int)(d >> sub) - (int)from;
                if (sub == SD_SHIFT) return min(max(b, 0), SBINS - 1);
                return (d >> in) == pre && (unsigned)b < (unsigned)SBINS ? b : -1;
            };
            if (!looked) each([&](const float (&v)[4], int i) {
                int at[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) at[e] = kept(v[e], i + e) ? bin(v[e]) : -1;
                if ((at[0] & at[1] & at[2] & at[3]) < 0) return;  // none of the four: all are -1
                u64 w[4];
                if (MASS) weights(v, {at[0] >= 0, at[1] >= 0, at[2] >= 0, at[3] >= 0}, w);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at[e] >= 0) {
                        atomicAdd(&s.n[at[e]], 1u);
                        if (MASS) {
                            const unsigned l = (unsigned)w[e], old = atomicAdd(&s.lo[at[e]], l);
                            const unsigned h = (unsigned)(w[e] >> 32) + (old + l < l ? 1u : 0u);
                            if (h) atomicAdd(&s.hi[at[e]], h);
                        }
                    }
            });
            if (!looked) join_bins<MASS>();
            const u64 m = MASS ? s.all_w[tid] : (u64)s.all_n[tid];
            if (MASS && level == 0) {
                const u64 inc = block_scan(s, m);
                if (tid == ST - 1) s.cut = inc;
                __syncthreads();
                *all = s.cut;
                want = prefix(p, *all);
            }
            const int b = looked ? s.found : reach(m, base, want);
            looked = false;
            if (b < 0) return 0;  // fewer entries than k: all are kept
            base = s.found_before;
            const unsigned n = s.all_n[b];
            if (level == 0 && whole) {  // everything down to this bin
                const u64 upto = block_scan(s, tid <= b ? s.all_n[tid] : 0u);
                if (tid == ST - 1) s.found_w = upto;
                __syncthreads();
                if (s.found_w <= SLIST && b < SBINS - 1) return (int)gather_to(b);
            }
            if (n <= SLIST) {
                // (a bin of images is a stretch of scores)
                const float from_x = by_image ? f32_from_ord(max(ohi - (((unsigned)b + 1u) << sub) + 1u, olo)) : -CUDART_INF_F;
                const float to_x = by_image ? f32_from_ord(ohi - ((unsigned)b << sub)) : CUDART_INF_F;
                // the look's bin: what the stretch has above it is added to the sums of what lies above the stretch
                const bool direct = MASS && seen == 1 && level == 1;
                const float end_x = direct ? split : to_x;
                u64 w_in = 0;
                unsigned n_in = 0;
                each([&](const float (&v)[4], int i) {
                    bool among[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) among[e] = v[e] >= from_x && v[e] <= end_x;
                    if (!(among[0] | among[1] | among[2] | among[3])) return;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!among[e]) continue;
                        const int at = kept(v[e], i + e) ? bin(v[e]) : -1;
                        among[e] = at == b;
                        if (direct && at >= 0 && at < b) w_in += weight(v[e]), ++n_in;
                    }
                    note(among, v, i);
                });
                if (direct) {
                    w_in = warp_sum(w_in);
                    n_in = __reduce_add_sync(0xffffffffu, n_in);
                    if (lane == 0) s.above_w[warp] += w_in, s.above_n[warp] += n_in;
                }
                deliver();
                if (rank == 0) {
                    const u64 mine = block_sort(s, fetch(), (int)n);
                    const u64 w = tid >= (int)n ? 0ull : (MASS ? weight_of(f32_from_ord(key_ord(mine))) : 1ull);
                    const u64 inc = block_scan(s, w) + base;
                    if (inc >= want && inc - w < want)
                        for (int r = 0; r < a.ctas; ++r) s_put(s_at(&s.cut, r), mine);
                }
                sync();
                keep_from(s.cut);
                if (direct) {  // and of the bin what is kept
                    if (tid < (int)s.slot_n[rank] && s.list[tid] >= s.cut) {
                        const u64 k = s.list[tid];
                        const int of = (int)(key_slot(k) - (unsigned)start) / wlen;
                        atomicAdd(&s.above_w[of], weight(f32_from_ord(key_ord(k))));
                        atomicAdd(&s.above_n[of], 1u);
                    }
                    __syncthreads();
                    summed = true;
                }
                return 0;
            }
            // too many: the next bits of the distance, where the bin is one value of the bits above
            if (!by_image && sub > 0 && (level > 0 || (b > 0 && b < SBINS - 1))) {
                in = sub;
                pre = from + (unsigned)b;
                sub = max(sub - 10, 0);
                from = pre << (in - sub);
                continue;
            }
            // the bits of the scores, between the least and the largest of the bin
            unsigned least = ~0u, most = 0;
            each([&](const float (&v)[4], int i) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (kept(v[e], i + e) && bin(v[e]) == b) {
                        const unsigned o = ord_from_f32(v[e]);
                        least = min(least, o), most = max(most, o);
                    }
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
                const float tied = f32_from_ord(olo);
                const u64 each_w = MASS ? weight_of(tied) : 1ull;
                const u64 need = (want - base + each_w - 1) / each_w;  // each_w > 0: the bin reaches the target
                if (need < n) {
                    const auto tie = [&](float v, int i) { return v == tied && kept(v, i); };
                    unsigned none;
                    sums<false>([&](const float (&v)[4], int i, bool (&k)[4]) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) k[e] = tie(v[e], i + e);
                    }, &none);
                    walk<false>(tie, need - 1);
                    if (tid == 0 && s.found >= 0)
                        for (int r = 0; r < a.ctas; ++r) s_put(s_at(&s.cut, r), key(tied, s.found));
                    sync();
                    keep_from(s.cut);
                } else
                    keep_from(max(thr, (u64)make_key(olo, ~0u)));
                return 0;
            }
            by_image = true;
            sub = 0;
            while (((ohi - olo) >> sub) >= SBINS) ++sub;
        }
    }
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(ST) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char s_raw[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(s_raw);
    const long long row = blockIdx.x / a.ctas;
    const int rank = blockIdx.x % a.ctas;  // the cluster is the row's CTAs, in order
    const int start = min(rank * a.seg, a.vocab);
    using R = Row<T, WIDE>;
    R w = {a, s, reinterpret_cast<T *>(s_raw + sizeof(SampleShared)), static_cast<const T *>(a.logits) + row * a.ld + start};
    constexpr int PER = R::PER;
    const int tid = w.tid = threadIdx.x, lane = w.lane = tid & 31, warp = w.warp = tid >> 5;
    w.rank = rank;
    w.start = start;
    w.len = min(a.seg, a.vocab - start);
    w.wlen = (int)round_up((w.len + SWARPS - 1) / SWARPS, PER);

    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float least_in = a.min_p ? a.min_p[row] : 0.0f;
    const float u = a.u[row];
    const bool bad = !(temp >= 0.0f) || p != p || least_in != least_in || u != u;
    if (temp == 0.0f) temp = 1.0f, k = 1;
    s.octave[tid >> 3][tid & 7] = exp2((tid >> 3) / 128.0) * (double)(1ull << a.unit_bits);  // as many as threads
    if (a.ctas > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");  // waited for before the first write to another CTA

    w.unit_bits = a.unit_bits;
    w.temp = temp;
    w.split = CUDART_INF_F;
    w.summed = false;
    w.octaves = 128.0 / (0.693147180559945309417232 * (double)temp);
    w.per_t = fminf(1.0f / temp, 3e38f);

    // ---- the row comes in; its largest score ----
    const int held = min(w.len, a.cap);
    float largest = -CUDART_INF_F;  // that this thread has seen; fmaxf passes over NaN
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(w.x) & 15) == 0) {
        const int vecs = w.len / PER, to_keep = held / PER;  // (cap is a multiple of PER)
        done = vecs * PER;
        constexpr int U = 4;
        for (int v0 = tid; v0 < vecs; v0 += ST * U) {
            uint4 q[U];
#pragma unroll
            for (int e = 0; e < U; ++e)
                if (v0 + e * ST < vecs) q[e] = reinterpret_cast<const uint4 *>(w.x)[v0 + e * ST];
#pragma unroll
            for (int e = 0; e < U; ++e)
                if (v0 + e * ST < vecs) {
                    if (v0 + e * ST < to_keep) reinterpret_cast<uint4 *>(w.data)[v0 + e * ST] = q[e];
                    const T *t = reinterpret_cast<const T *>(&q[e]);
#pragma unroll
                    for (int i = 0; i < PER; ++i) largest = fmaxf(largest, Elem<T>::get(t[i]));
                }
        }
    }
    for (int i = done + tid; i < w.len; i += ST) {
        const T t = w.x[i];
        if (i < held) w.data[i] = t;
        largest = fmaxf(largest, Elem<T>::get(t));
    }
    for (int i = held + tid; i < (int)round_up(held, PER); i += ST) w.data[i] = Elem<T>::put(CUDART_NAN_F);
    const unsigned own = ord_from_f32(largest);
    unsigned top = __reduce_max_sync(0xffffffffu, own);
    if (lane == 0) s.warp_n[warp] = top;
    __syncthreads();
    if constexpr (WIDE) {
        // No entry weighs more than the largest that its thread has seen, so the weight of the CTA's entries is at most `each` times the
        // sum of those.  In 2^-20, rounded up, with 1 % for the common factor of the weights and the roundings here.
        top = __reduce_max_sync(0xffffffffu, s.warp_n[lane]);
        const u64 each = (u64)(w.len / ST + PER + 1);  // entries of a thread, as they came in
        u64 most = 0;
        if (own > kNegInf) most = __float2ull_ru(w.lighter(largest, f32_from_ord(top)) * (1.01f * 1048576.0f)) + 1;
        most = warp_sum(most) * each;
        if (lane == 0) s.warp_w[warp] = most;
        __syncthreads();
    }
    if (a.ctas > 1) asm volatile("barrier.cluster.wait;" ::: "memory");  // every CTA of the cluster runs
    if (warp == 0) {
        top = __reduce_max_sync(0xffffffffu, s.warp_n[lane]);
        if (lane < a.ctas) s_put(s_at(&s.slot_top[rank], lane), top);
        if constexpr (WIDE) {
            const u64 most = warp_sum(s.warp_w[lane]);
            if (lane < a.ctas) s_put(s_at(&s.slot_v[rank], lane), most);
        }
    }
    w.sync();
    for (int r = 0; r < a.ctas; ++r) top = max(top, s.slot_top[r]);
    if (bad || top <= kNegInf) {  // the whole cluster agrees
        if (rank == 0 && tid == 0) {
            a.ids[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
            if (a.kept) a.kept[row] = 0;
        }
        return;  // nothing is written to this CTA any more
    }
    w.top = f32_from_ord(top);
    w.top_wide = (double)w.top;
    w.whole = 6755399441055744.0 - rint(w.top_wide * w.octaves);
    // 62 octaves down a weight rounds to 0 (F <= 49).  Where the next lower float32 is further down than that, nothing but the
    // largest score weighs; else `bottom` is 62 to 124 octaves down, or the lowest score there is.
    const double deep = 62.0 * 0.693147180559945309417232 * (double)temp;
    w.alone = !(w.top_wide - (double)nextafterf(w.top, -CUDART_INF_F) < deep);  // true for +infinity
    w.bottom = __double2float_rd(fmax(w.top_wide - deep, -(double)FLT_MAX));
    if constexpr (WIDE) {
        u64 most = 0;  // every CTA's bound, which is in weights of its own largest score, in the row's
        if (lane < a.ctas) most = __float2ull_ru((float)s.slot_v[lane] * w.lighter(f32_from_ord(s.slot_top[lane]), w.top)) + 1;
        most = warp_sum(most);
        w.unit_bits = max(a.unit_bits, min(62 + 20 - (64 - __clzll((long long)most)), 49));
        s.octave[tid >> 3][tid & 7] *= (double)(1ull << (w.unit_bits - a.unit_bits));
        __syncthreads();
    }
    w.floor = 0ull;
    if (least_in > 0.0f) {
        if (warp == 0) {
            const u64 f = w.lowest(fminf(least_in, 1.0f));
            if (lane == 0) s.floor = f;
        }
        __syncthreads();
        w.floor = s.floor;
    }
    w.keep_from(make_key(kNegInf + 1, 0xffffffffu - 1u));

    // ---- few candidates ----
    int n = 0;
    u64 all = 0;
    if (k > 0 && k <= SLIST / 2) {
        w.template clear_bins<false>();
        if (own > kNegInf) atomicAdd(&s.n[R::first_bin(w.distance(f32_from_ord(own)))], 1u);
        w.template join_bins<false>();
        const int b = w.reach(s.all_n[tid], 0, (u64)k);
        if (b >= 0 && b < SBINS - 1) n = (int)w.gather_to(b);
        if (n > SLIST) n = 0;
    }
    // ---- the cuts ----
    if (n == 0) {
        const bool by_count = k > 0 && k < a.vocab;
        if (by_count) w.template cut<false>(k, 1.0f, false, &all);
        if (p < 1.0f) n = w.template cut<true>(0, p, !by_count, &all);
    }
    if (n > 0) {
        if (rank == 0) w.finish(row, n, k, p, u, all);
        if (a.ctas > 1) w.sync();  // the others' shared memory is not needed any more, but was read above
        return;
    }

    // ---- the draw ----
    unsigned count = 0;
    const auto keep = [&](float v, int i) { return w.kept(v, i); };
    if (w.floor > w.thr) w.split = CUDART_INF_F, w.summed = false;  // min-p cuts higher: the sums above the other cut are of no use
    w.keep_from(max(w.thr, w.floor));
    if (w.summed) {
        all = w.join_sums(s.above_w[warp]);
        if (lane == 0) count = s.above_n[warp];
    } else
        all = w.template sums<true>([&](const float (&v)[4], int i, bool (&k)[4]) {
            w.kept4(v, i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = k[e] && !(v[e] > w.split);  // what lies above has been summed
        }, &count);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) s.warp_n[warp] = count;
    w.template walk<true>(keep, R::aim(u, all));
    __syncthreads();
    if (s.found >= 0 && tid == 0) {
        a.ids[row] = start + s.found;
        if (a.probs) a.probs[row] = (float)((double)s.found_w / (double)all);
    }
    if (a.kept) {
        if (warp == 0) {
            const unsigned c = __reduce_add_sync(0xffffffffu, s.warp_n[lane]);
            if (lane == 0) s_put(s_at(&s.slot_b[rank], 0), c);
        }
        w.sync();
        if (rank == 0 && tid == 0) {
            unsigned c = 0;
            for (int r = 0; r < a.ctas; ++r) c += s.slot_b[r];
            a.kept[row] = (int)c;
        }
    }
}

template <typename T, bool WIDE>
static int sample_launch(SampleArgs a, long long rows, int device, cudaStream_t st) {
    constexpr size_t kSmem = 227 * 1024;
    constexpr int kHold = (int)((kSmem - sizeof(SampleShared)) / sizeof(T)) & ~63;
    static OncePerDevice asked;
    static int fit[kMaxDevices][SMAX_CTAS + 1];  // clusters of so many full CTAs that run at the same time
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(ST);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LK_TRY(asked.run(device, [&] {
        LK_CUDA(cudaFuncSetAttribute((const void *)k_sample<T, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        LK_CUDA(cudaFuncSetAttribute((const void *)k_sample<T, WIDE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cfg.dynamicSmemBytes = kSmem;
        for (int c = 1; c <= SMAX_CTAS; ++c) {
            attr[0].val.clusterDim.x = (unsigned)c;
            cfg.gridDim = dim3((unsigned)c);
            if (cudaOccupancyMaxActiveClusters(&fit[device][c], k_sample<T, WIDE>, &cfg) != cudaSuccess) fit[device][c] = 0;
        }
        cudaGetLastError();
        return 0;
    }));
    // The number of CTAs to a row that finishes first: clusters run in waves, a CTA's time is its entries (those past what
    // its shared memory holds cost more) and its meetings.
    double least = 1e300;
    for (int c = 1; c <= SMAX_CTAS; ++c) {
        if (c > 1 && fit[device][c] < 1) continue;
        const double waves = (double)((rows + std::max(fit[device][c], 1) - 1) / std::max(fit[device][c], 1));
        const double seg = (double)((a.vocab + c - 1) / c);
        const double cost = waves * (SAMPLE_ENTRY_NS * seg + SAMPLE_AWAY_NS * std::max(0.0, seg - kHold) + (c > 1 ? SAMPLE_MEET_NS : 0.0) +
                                     (c > 8 ? SAMPLE_WIDE_NS : 0.0) + SAMPLE_CTA_NS);
        if (cost < least) least = cost, a.ctas = c;
    }
    a.seg = (int)round_up((a.vocab + a.ctas - 1) / a.ctas, 64);
    a.cap = std::min(a.seg, kHold);
    attr[0].val.clusterDim.x = (unsigned)a.ctas;
    cfg.gridDim = dim3((unsigned)(rows * a.ctas));
    cfg.dynamicSmemBytes = sizeof(SampleShared) + (size_t)a.cap * sizeof(T);
    cfg.stream = st;
    return launch_cfg("lk_sample", k_sample<T, WIDE>, cfg, a);
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
                    reinterpret_cast<long long *>(d_ids), d_probs, d_kept, std::min(62 - bits, 49)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = vocab > kWide;
    if (dtype == LK_F32) return wide ? sample_launch<float, true>(a, rows, device, st) : sample_launch<float, false>(a, rows, device, st);
    if (dtype == LK_F16) return wide ? sample_launch<__half, true>(a, rows, device, st) : sample_launch<__half, false>(a, rows, device, st);
    return wide ? sample_launch<__nv_bfloat16, true>(a, rows, device, st) : sample_launch<__nv_bfloat16, false>(a, rows, device, st);
}
