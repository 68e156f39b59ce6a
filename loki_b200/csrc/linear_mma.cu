// Matrix product of rows with rows on the tensor cores (tcgen05.mma, accumulators in tensor memory), the
// scales, bias, activation and residual in its epilogue.
//
// The rows of w take the M side of the MMA (tensor-memory lanes), the rows of a its N side (columns): a
// tile is 128 rows of w per CTA and `mt` rows of a, mt from 16 (single tokens: the MMA's smallest N) to 256.
// One kernel thus serves one token and thousands, and an epilogue thread owns one column j of the
// result: its scale and bias are two registers, and the 32 threads of a warp read the residual and write
// the result 32 neighbours at a time, with no staging.
//
// Both operands arrive as [rows x 128 bytes] slices of K by TMA (128-byte swizzle), rows and columns past
// the ends as zeros, through a ring of stages; 128 bytes are 128 int8 or 64 16-bit elements, four
// MMAs either way.  Roles of a CTA: warp 0 issues the copies, warp 1 the MMAs, warps 2-17 are the epilogue (two
// accumulators: a tile's epilogue runs under the next tile's MMAs).
//
// Two forms.  PAIR: two CTAs of a cluster share every MMA (cta_group::2, 256 rows of w), each loads its
// own 128 rows of w and half the rows of a.  Single: one CTA per tile, and where there are too few tiles
// to fill the GPU a cluster of `split` CTAs shares one tile's K: each sums its part and sends every
// other CTA its share of the columns straight from registers into shared memory (st.async, counted on the owner's
// barrier), where the parts are added in rank order (the result does not depend on timing) and finished.  No workspace, no
// atomics, and the cluster meets only once, while the first copies are under way.
//
// Every wait is bounded; a CTA that gives up raises g_linear_failed, which lk_ops_status reports.
#include <cstddef>
#include <type_traits>

#include "linear.cuh"
#include "tensor5.cuh"

namespace lk {

constexpr int LW = 128;             // rows of w per CTA (tensor-memory lanes)
constexpr int LSLICE = 128;         // bytes of K per stage: one swizzle row
constexpr int LW_BYTES = LW * LSLICE;
constexpr int LEPI_WARPS = 16;      // four per tensor-memory quadrant, 16 columns of a tile at a time each
constexpr int LTHREADS = 64 + LEPI_WARPS * 32;
// A long stream, 8,192 x 18 KB slices of an m = 8 product: 26.4 us with 8 stages, 27.6 with 6, 28.4 with 12.  Nothing else was measured: for one
// tile of few slices more would fit (11 with 32 rows of a), and the latency that linear_plan counts per stage is paid twice there.
constexpr int LMAX_STAGES = 8;
constexpr int LCHUNK = 16;          // columns an epilogue thread holds at a time

static __device__ unsigned g_linear_failed;  // a bounded wait ran out on this device

struct LinearTiles {
    int mt;              // rows of a per tile
    int stages, split;
    int slices;          // K slices of 128 bytes
    int tiles_m, tiles_n, band;
    long long tiles;
    unsigned idesc;
    unsigned columns;    // tensor memory to allocate
    bool w_once;         // every row of w is read by one CTA only, and all of w is more than L2 would keep
};

// Place of tile t: bands of `band` tiles of w's rows, through which the tiles of a's rows run.  Where w is the smaller operand a
// band as wide as w keeps it in L2 and reads a once: 8,192 x 4,096 x 4,096 bf16, sustained: 228 us with bands of 1, 216 of 8, 208 of
// all 16.  Else bands of 8, which also serve an `a` that is too large to stay (4,096 x 8,192 x 4,096 int8: 102.5 us with bands of 1,
// 103.7 of 8, 105.5 of 16).  These two sizes are all that was timed.
__device__ __forceinline__ void tile_at(const LinearTiles &g, long long t, int &tn, int &tm) {
    const long long per = (long long)g.band * g.tiles_m;
    const int band = (int)(t / per), r = (int)(t - band * per);
    const int width = min(g.band, g.tiles_n - band * g.band);
    tm = r / width;
    tn = band * g.band + r - tm * width;
}

struct LinearShared {
    unsigned long long full[LMAX_STAGES], empty[LMAX_STAGES], acc_full[2], acc_empty[2], joined;
    alignas(16) float sa[2][256];  // the scales of a tile's rows of a, per accumulator
    unsigned tmem_base;
    int failed;
};

static_assert(offsetof(LinearShared, sa) % 16 == 0, "read four at a time");

// 2-D tiled TMA load into this CTA's shared memory, counted on `bar` (PAIR: the leader's).
template <bool PAIR>
__device__ __forceinline__ void l_load(unsigned dst, const CUtensorMap *tm, int x, int y, unsigned bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<unsigned long long>(tm)), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<unsigned long long>(tm)), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

// The same, the lines first to go from L2: for what is read once.
__device__ __forceinline__ void l_load_once(unsigned dst, const CUtensorMap *tm, int x, int y, unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
        "l"(reinterpret_cast<unsigned long long>(tm)), "r"(x), "r"(y), "r"(bar), "l"(0x12F0000000000000ull)
        : "memory");
}

__device__ __forceinline__ unsigned l_at(unsigned local, int rank) {  // a shared-memory address as it sits in CTA `rank`
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
// Words to another CTA's shared memory, counted on its barrier.
__device__ __forceinline__ void l_send(unsigned to, unsigned a, unsigned b, unsigned c, unsigned d, unsigned bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar) : "memory");
}
__device__ __forceinline__ void l_send(unsigned to, unsigned a, unsigned b, unsigned bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to), "r"(a), "r"(b), "r"(bar) : "memory");
}

template <bool PAIR, bool I8>
__device__ __forceinline__ void l_mma(unsigned d, unsigned long long dw, unsigned long long da, unsigned idesc, bool accumulate) {
    const unsigned acc = accumulate ? 1u : 0u;
#define LK_MMA(GROUP, KIND)                                                              \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                       \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" \
                 ::"r"(d), "l"(dw), "l"(da), "r"(idesc), "r"(acc) : "memory")
    if constexpr (PAIR && I8) LK_MMA("2", "i8");
    else if constexpr (PAIR) LK_MMA("2", "f16");
    else if constexpr (I8) LK_MMA("1", "i8");
    else LK_MMA("1", "f16");
#undef LK_MMA
}

// Arrive on `bar` (PAIR: at its address in both CTAs) once the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void l_commit(unsigned long long *bar) {
    if constexpr (PAIR) g_mma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(g_smem(bar)) : "memory");
}

__device__ __forceinline__ void l_tmem_ld16(unsigned taddr, unsigned (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

template <bool I8>
__device__ __forceinline__ float l_sum(unsigned bits) {
    if constexpr (I8) return (float)(int)bits;
    else return __uint_as_float(bits);
}

template <bool PAIR, bool I8, typename Out>
__global__ void __launch_bounds__(LTHREADS, 1)
k_linear_mma(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const LinearArgs p, const LinearTiles g) {
    constexpr int CG = PAIR ? 2 : 1;
    extern __shared__ unsigned char l_raw[];
    // 1024-byte alignment: the swizzle pattern is a function of the shared-memory address
    unsigned char *smem = l_raw + ((1024u - (g_smem(l_raw) & 1023u)) & 1023u);
    const int a_bytes = g.mt / CG * LSLICE;
    unsigned char *sm_w = smem;                                    // [stages][128 rows][128 B]
    unsigned char *sm_a = sm_w + (size_t)g.stages * LW_BYTES;      // [stages][mt / CG rows][128 B]
    const bool joined = !PAIR && g.split > 1;
    unsigned *sm_parts = reinterpret_cast<unsigned *>(sm_a + (size_t)g.stages * a_bytes);  // split: [CTA][columns / w][128][w] of this CTA's columns
    LinearShared *ctl = reinterpret_cast<LinearShared *>(sm_parts + (joined ? g.mt * LW : 0));

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = PAIR || g.split > 1 ? (int)g_cta_rank() : 0;
    const int cta_of = PAIR ? rank : 0;          // which half of the pair's tile
    const int part_of = PAIR ? 0 : rank;         // which part of K
    const int per = PAIR ? 2 : g.split;          // CTAs per tile
    const long long first = blockIdx.x / per, step = gridDim.x / per;
    const int s0 = (int)((long long)g.slices * part_of / (PAIR ? 1 : g.split));
    const int s1 = (int)((long long)g.slices * (part_of + 1) / (PAIR ? 1 : g.split));

    const int early = PAIR ? 0 : min(g.stages, s1 - s0);  // slices of the first tile that need no free stage waited for

    if (tid == 0) {
        for (int i = 0; i < g.stages; ++i) {
            g_mbar_init(&ctl->full[i], 1);
            g_mbar_init(&ctl->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            g_mbar_init(&ctl->acc_full[i], 1);
            g_mbar_init(&ctl->acc_empty[i], CG * LEPI_WARPS);
        }
        ctl->failed = 0;
        if (joined) g_mbar_init(&ctl->joined, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (joined) g_mbar_expect_tx(&ctl->joined, (unsigned)(g.mt * LW * 4));
        if (!PAIR && first < g.tiles) {  // the first stages are on their way while the CTA sets itself up
            int tn, tm;
            tile_at(g, first, tn, tm);
            const int yw = tn * LW, ya = tm * g.mt;
            for (int i = 0; i < early; ++i) {
                g_mbar_expect_tx(&ctl->full[i], (unsigned)(LW_BYTES + a_bytes));
                if (g.w_once) l_load_once(g_smem(sm_w + (size_t)i * LW_BYTES), &tm_w, (s0 + i) * LSLICE, yw, g_smem(&ctl->full[i]));
                else l_load<PAIR>(g_smem(sm_w + (size_t)i * LW_BYTES), &tm_w, (s0 + i) * LSLICE, yw, g_smem(&ctl->full[i]));
                l_load<PAIR>(g_smem(sm_a + (size_t)i * a_bytes), &tm_a, (s0 + i) * LSLICE, ya, g_smem(&ctl->full[i]));
            }
        }
    }
    if (warp == 1) {
        __syncwarp();
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem(&ctl->tmem_base)), "r"(g.columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem(&ctl->tmem_base)), "r"(g.columns) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) g_pair_sync();  // the partner's barriers exist before anything is signalled across
    // so do the others'; waited for before the first word is sent.  Relaxed: the fence behind the barriers' set-up is all that
    // has to be seen, and a release by every thread held up the first MMAs
    if (joined) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = ctl->tmem_base;
    volatile int *failed = &ctl->failed;

    if (warp == 0) {
        // ------------------------------ copies ------------------------------
        int stage = 0;
        unsigned phase = 0;
        bool ok = true;
        for (long long t = first; ok && t < g.tiles; t += step) {
            int tn, tm;
            tile_at(g, t, tn, tm);
            const int yw = tn * LW * CG + cta_of * LW;
            const int ya = tm * g.mt + cta_of * (g.mt / CG);
            for (int s = s0; s < s1; ++s) {
                if (t == first && s - s0 < early) {
                    // already asked for.  Its stage must not be waited for either: it may have been used and freed by
                    // now, and the wait would be for the phase after that
                    if (++stage == g.stages) stage = 0, phase ^= 1u;
                    continue;
                }
                ok = g_mbar_wait_warp(&ctl->empty[stage], phase ^ 1u, failed);
                if (!ok) break;
                if (g_elect_one()) {
                    const unsigned bar = PAIR ? g_leader_addr(g_smem(&ctl->full[stage])) : g_smem(&ctl->full[stage]);
                    if (cta_of == 0) g_mbar_expect_tx(&ctl->full[stage], (unsigned)(CG * (LW_BYTES + a_bytes)));
                    if (!PAIR && g.w_once) l_load_once(g_smem(sm_w + (size_t)stage * LW_BYTES), &tm_w, s * LSLICE, yw, bar);
                    else l_load<PAIR>(g_smem(sm_w + (size_t)stage * LW_BYTES), &tm_w, s * LSLICE, yw, bar);
                    l_load<PAIR>(g_smem(sm_a + (size_t)stage * a_bytes), &tm_a, s * LSLICE, ya, bar);
                }
                __syncwarp();
                if (++stage == g.stages) stage = 0, phase ^= 1u;
            }
        }
    } else if (warp == 1 && cta_of == 0) {
        // ------------------------------ MMAs ------------------------------
        const unsigned long long dw0 = g_smem_desc(g_smem(sm_w)), da0 = g_smem_desc(g_smem(sm_a));
        int stage = 0, acc = 0;
        unsigned phase = 0, acc_phase = 0;
        bool ok = true;
        for (long long t = first; ok && t < g.tiles; t += step) {
            ok = g_mbar_wait_warp(&ctl->acc_empty[acc], acc_phase ^ 1u, failed);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned d = tmem + (unsigned)(acc * g.mt);
            for (int s = s0; s < s1; ++s) {
                ok = g_mbar_wait_warp(&ctl->full[stage], phase, failed);
                if (!ok) break;
                // the start-address field counts 16-byte units
                const unsigned long long dw = dw0 + (unsigned long long)(stage * (LW_BYTES >> 4));
                const unsigned long long da = da0 + (unsigned long long)(stage * (a_bytes >> 4));
                if (g_elect_one()) {
#pragma unroll
                    for (int q = 0; q < LSLICE / 32; ++q)  // 32 bytes of K per MMA
                        l_mma<PAIR, I8>(d, dw + (unsigned long long)(2 * q), da + (unsigned long long)(2 * q), g.idesc, s != s0 || q != 0);
                    l_commit<PAIR>(&ctl->empty[stage]);
                }
                __syncwarp();
                if (++stage == g.stages) stage = 0, phase ^= 1u;
            }
            if (!ok) break;
            if (g_elect_one()) l_commit<PAIR>(&ctl->acc_full[acc]);
            __syncwarp();
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
    } else if (warp >= 2) {
        // ------------------------------ epilogue ------------------------------
        const int quad = warp & 3, part = (warp - 2) >> 2;  // the lanes a warp may read; the chunks it takes
        const int et = tid - 64;
        const long long ldr = p.ldr * (long long)sizeof(Out), ldo = p.ldo * (long long)sizeof(Out);
        bool epi_ok = true;
        int acc = 0;
        unsigned acc_phase = 0;
        for (long long t = first; t < g.tiles; t += step) {
            int tn, tm;
            tile_at(g, t, tn, tm);
            const long long j = (long long)tn * (LW * CG) + cta_of * LW + quad * 32 + lane;
            const long long i0 = (long long)tm * g.mt;
            const bool live = j < p.n;
            const bool whole = i0 + g.mt <= p.m && (j | 31) < p.n;  // this warp's share lies inside the result
            const float sw = live ? scale_of(p.w_scales, j) : 0.0f;
            const float bias = live && p.bias != nullptr ? Elem<Out>::get(static_cast<const Out *>(p.bias)[j]) : 0.0f;
            const char *res = static_cast<const char *>(p.residual) + i0 * ldr + j * (long long)sizeof(Out);
            char *out = static_cast<char *>(p.out) + i0 * ldo + j * (long long)sizeof(Out);
            // the residual of the chunk that comes next, fetched while the one before it is worked on (the first
            // while the MMAs still run)
            Out r[LCHUNK];
            const auto fetch = [&](int c) {
                const char *q = res + c * ldr;
#pragma unroll
                for (int u = 0; u < LCHUNK; ++u, q += ldr)
                    if (whole || (live && i0 + c + u < p.m)) r[u] = *reinterpret_cast<const Out *>(q);
            };
            if (!joined) {
                // the tile before last, which read this buffer, is behind every warp's last arrival at this barrier
                if (p.a_scales != nullptr && et < g.mt) ctl->sa[acc][et] = i0 + et < p.m ? p.a_scales[i0 + et] : 0.0f;
                if (p.residual != nullptr && part * LCHUNK < g.mt) fetch(part * LCHUNK);
                asm volatile("bar.sync 1, %0;" ::"n"(LEPI_WARPS * 32) : "memory");
            }
            if (!g_mbar_wait_warp(&ctl->acc_full[acc], acc_phase, failed)) epi_ok = false;
            if (!epi_ok) {
                if (joined) asm volatile("barrier.cluster.wait;" ::: "memory");
                // the other warps of the epilogue may be waiting at the barrier above: stay with them to the last tile
                if (++acc == 2) acc = 0, acc_phase ^= 1u;
                continue;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (joined) asm volatile("barrier.cluster.wait;" ::: "memory");
            for (int c = part * LCHUNK; c < g.mt; c += 4 * LCHUNK) {
                unsigned v[LCHUNK];
                l_tmem_ld16(tmem + (unsigned)(acc * g.mt + c) + ((unsigned)(quad * 32) << 16), v);
                float rx[LCHUNK], x[LCHUNK];
                if (p.residual != nullptr && !joined) {
#pragma unroll
                    for (int u = 0; u < LCHUNK; ++u) rx[u] = Elem<Out>::get(r[u]);
                    if (c + 4 * LCHUNK < g.mt) fetch(c + 4 * LCHUNK);
                }
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (joined) {  // this CTA's part of the sums, to the CTAs whose columns these are
                    const int own = g.mt / g.split, n = quad * 32 + lane;
                    if (own >= 4) {
#pragma unroll
                        for (int u = 0; u < LCHUNK; u += 4) {
                            const int to = (c + u) / own, at = ((part_of * own + (c + u) % own) >> 2) * LW + n;
                            l_send(l_at(g_smem(sm_parts + 4 * at), to), v[u], v[u + 1], v[u + 2], v[u + 3], l_at(g_smem(&ctl->joined), to));
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < LCHUNK; u += 2) {
                            const int to = (c + u) / own, at = ((part_of * own + (c + u) % own) >> 1) * LW + n;
                            l_send(l_at(g_smem(sm_parts + 2 * at), to), v[u], v[u + 1], l_at(g_smem(&ctl->joined), to));
                        }
                    }
                    continue;
                }
                if (p.a_scales != nullptr) {
#pragma unroll
                    for (int u = 0; u < LCHUNK; u += 4) {
                        const float4 f = *reinterpret_cast<const float4 *>(&ctl->sa[acc][c + u]);
                        x[u] = fmaf(l_sum<I8>(v[u]), f.x * sw, bias);
                        x[u + 1] = fmaf(l_sum<I8>(v[u + 1]), f.y * sw, bias);
                        x[u + 2] = fmaf(l_sum<I8>(v[u + 2]), f.z * sw, bias);
                        x[u + 3] = fmaf(l_sum<I8>(v[u + 3]), f.w * sw, bias);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < LCHUNK; ++u) x[u] = fmaf(l_sum<I8>(v[u]), sw, bias);
                }
                activate_all<std::is_same<Out, float>::value>(p.act, x);
                if (p.residual != nullptr) {
#pragma unroll
                    for (int u = 0; u < LCHUNK; ++u) x[u] += rx[u];
                }
                char *q = out + c * ldo;
                if (whole) {
#pragma unroll
                    for (int u = 0; u < LCHUNK; ++u, q += ldo) *reinterpret_cast<Out *>(q) = Elem<Out>::put(x[u]);
                } else {
#pragma unroll
                    for (int u = 0; u < LCHUNK; ++u, q += ldo)
                        if (live && i0 + c + u < p.m) *reinterpret_cast<Out *>(q) = Elem<Out>::put(x[u]);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (PAIR) g_mbar_arrive_leader(&ctl->acc_empty[acc]);
                else g_mbar_arrive(&ctl->acc_empty[acc]);
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
        }
    }
    // ------------------------------ joining the parts of K ------------------------------
    if (joined && warp >= 2) {  // one tile per cluster; this CTA's columns are mt / split of it
        const int own = g.mt / g.split, w = own >= 4 ? 4 : 2, items = own / w * LW;
        int tn, tm;
        tile_at(g, first, tn, tm);
        const long long j0 = (long long)tn * LW, i0 = (long long)tm * g.mt + part_of * own;
        bool ok = true, waited = false;
        for (int e = tid - 64; e < items; e += LEPI_WARPS * 32) {  // one column of the result, w rows of it
            const int n = e % LW;
            const long long i = i0 + e / LW * w, j = j0 + n;
            const bool live = j < p.n;
            // the epilogue's inputs are on their way while the parts are
            const float sw = live ? scale_of(p.w_scales, j) : 0.0f;
            const float bias = live && p.bias != nullptr ? Elem<Out>::get(static_cast<const Out *>(p.bias)[j]) : 0.0f;
            float sa[4], r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool there = live && u < w && i + u < p.m;
                sa[u] = there ? scale_of(p.a_scales, i + u) : 0.0f;
                r[u] = there && p.residual != nullptr ? Elem<Out>::get(static_cast<const Out *>(p.residual)[(i + u) * p.ldr + j]) : 0.0f;
            }
            if (!waited) ok = g_mbar_wait(&ctl->joined, 0u, failed), waited = true;
            if (!ok) break;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            int whole[4] = {0, 0, 0, 0};
            for (int q = 0; q < g.split; ++q) {
                unsigned v[4] = {0u, 0u, 0u, 0u};
                if (w == 4) {
                    const uint4 f = *reinterpret_cast<const uint4 *>(sm_parts + 4 * ((q * own >> 2) * LW + e));
                    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2 *>(sm_parts + 2 * ((q * own >> 1) * LW + e));
                    v[0] = f.x, v[1] = f.y;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if constexpr (I8) whole[u] += (int)v[u];
                    else x[u] += __uint_as_float(v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = fmaf(I8 ? (float)whole[u] : x[u], sa[u] * sw, bias);
            activate_all<std::is_same<Out, float>::value>(p.act, x);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (live && u < w && i + u < p.m)
                    static_cast<Out *>(p.out)[(i + u) * p.ldo + j] = Elem<Out>::put(p.residual != nullptr ? x[u] + r[u] : x[u]);
        }
        // whoever had nothing to finish waits too: this CTA's shared memory is written to until all parts are here
        if (!waited) g_mbar_wait(&ctl->joined, 0u, failed);
    }
    if (joined && warp < 2) asm volatile("barrier.cluster.wait;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (joined && ctl->failed != 0) {
        // This CTA did not wait for the others' parts, and one of them may still be on its way to sending its own here.  The barrier opens
        // when the other CTAs' threads have come here too or, as those that did not fail, have exited; all their waits are bounded.
        asm volatile("barrier.cluster.arrive;" ::: "memory");
        asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    if (tid == 0 && ctl->failed != 0) {
        atomicExch(&g_linear_failed, 1u);
        // copies this CTA issued may still be landing in its shared memory: give them time before it is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) {}
    }
    if (PAIR) g_pair_sync();  // nothing of the partner is still aimed at this CTA's barriers or tensor memory
    if (warp == 1) {
        __syncwarp();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.columns) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.columns) : "memory");
    }
}

bool linear_mma_reads(const LinearArgs &p, int dtype) {
    const int eb = type_bytes(dtype);
    const auto reads = [&](const void *base, long long rows, long long ld) {
        return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (rows == 1 || (ld * eb % 16 == 0 && ld * eb < (1ll << 40)));
    };
    return p.k > 0 && reads(p.a, p.m, p.lda) && reads(p.w, p.n, p.ldw);
}

struct LinearPlan {
    bool pair;
    int mt, split;
};

// Clusters of 2, 4 and 8 full CTAs that run at the same time on a device, asked once.
struct ClusterRoom {
    int of[9];
};
static int cluster_room(int device, const ClusterRoom **out) {
    static OncePerDevice once;
    static ClusterRoom rooms[kMaxDevices];
    ClusterRoom &r = rooms[device];
    LK_TRY(once.run(device, [&] {
        const void *f = (const void *)k_linear_mma<false, true, float>;
        LK_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.blockDim = dim3(LTHREADS);
        cfg.dynamicSmemBytes = 227 * 1024;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        r.of[1] = sm_count(device);
        for (int c = 2; c <= 8; c *= 2) {
            attr[0].val.clusterDim.x = (unsigned)c;
            cfg.gridDim = dim3((unsigned)c);
            if (cudaOccupancyMaxActiveClusters(&r.of[c], f, &cfg) != cudaSuccess) r.of[c] = 0;
        }
        cudaGetLastError();
        return 0;
    }));
    *out = &r;
    return 0;
}

// Stages of a ring beside the parts of K that arrive from the cluster.
static int ring_stages(int mt, int cg, int split) {
    return std::min((226 * 1024 - (int)sizeof(LinearShared) - 1024 - (split > 1 ? mt * LW * 4 : 0)) / (LW_BYTES + mt / cg * LSLICE), LMAX_STAGES);
}

// The tile that finishes first, by an account of one CTA's clocks whose constants were fitted to 110 shapes (m 1 to 1,024,
// five n x k, int8 and bf16) with every tile timed; over them the choice costs 0.2 % against the best tile, 4 % at worst.  Outside them
// (m to 8,192, k to 65,536) it is an extrapolation.
// A slice of K: its MMAs (0.62 clocks per row of a), its bytes at 58 per clock and SM and 5,456 for all CTAs together, and the
// 4,058 clocks from asking for a slice to having it, shared by the stages.  A tile's epilogue, 31 clocks per row of a, runs under
// the next tile's slices; the last one shows.  Joining parts of K costs 4,305 clocks and 16 per row of a.
static LinearPlan linear_plan(long long m, long long n, int slices, const ClusterRoom &room) {
    LinearPlan best = {false, 16, 1};
    double least = 1e300;
    const auto offer = [&](bool pair, int mt, int split) {
        const int cg = pair ? 2 : 1, per = cg * split;
        const long long tiles = ((m + mt - 1) / mt) * ((n + LW * cg - 1) / (LW * cg));
        if (room.of[per] < 1 || (split > 1 && (tiles > room.of[per] || split > slices))) return;
        const int stages = ring_stages(mt, cg, split);
        if (stages < 1) return;
        const double waves = (double)((tiles + room.of[per] - 1) / room.of[per]);
        const double bytes = LW_BYTES + mt / cg * LSLICE, active = (double)std::min<long long>(tiles * per, room.of[1]);
        const double slice = std::max(std::max(0.62 * mt, 4058.0 / stages), std::max(bytes / 58.0, active * bytes / 5456.0));
        const double main = (slices + split - 1) / split * slice, epilogue = 31.0 * mt / split;
        const double cost = waves * (waves > 1.0 ? std::max(main, epilogue) : main) + epilogue + (split > 1 ? 4305.0 + 16.0 * mt : 0.0);
        if (cost < least) least = cost, best = {pair, mt, split};
    };
    for (int mt = 16; mt <= 256; mt *= 2) {
        if (mt >= 2 * m && mt > 16) break;  // a smaller tile holds all rows
        for (int split = 1; split <= 8; split *= 2) offer(false, mt, split);
        if (mt >= 128) offer(true, mt, 1);
    }
    return best;
}

template <bool PAIR, bool I8, typename Out>
static int mma_launch(const CUtensorMap &tw, const CUtensorMap &ta, const LinearArgs &p, const LinearTiles &g, int device, int sms, cudaStream_t st) {
    constexpr int CG = PAIR ? 2 : 1;
    static OncePerDevice sized;
    const size_t smem = (size_t)g.stages * (LW_BYTES + g.mt / CG * LSLICE) + (g.split > 1 ? g.mt * LW * 4 : 0) + sizeof(LinearShared) + 1024;
    LK_TRY(sized.run(device, [] {
        LK_CUDA(cudaFuncSetAttribute((const void *)k_linear_mma<PAIR, I8, Out>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        return 0;
    }));
    const int per = PAIR ? 2 : g.split;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min<long long>(g.tiles, std::max(1, sms / per)) * per));
    cfg.blockDim = dim3(LTHREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)per;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = per > 1 ? 1 : 0;
    return launch_cfg("lk_linear", k_linear_mma<PAIR, I8, Out>, cfg, tw, ta, p, g);
}

template <bool PAIR, bool I8>
static int mma_out(const CUtensorMap &tw, const CUtensorMap &ta, const LinearArgs &p, const LinearTiles &g, int device, int sms, cudaStream_t st) {
    if (p.out_type == LK_F32) return mma_launch<PAIR, I8, float>(tw, ta, p, g, device, sms, st);
    if (p.out_type == LK_F16) return mma_launch<PAIR, I8, __half>(tw, ta, p, g, device, sms, st);
    return mma_launch<PAIR, I8, __nv_bfloat16>(tw, ta, p, g, device, sms, st);
}

int linear_mma_launch(const LinearArgs &p, int dtype, int device, cudaStream_t st) {
    const int eb = type_bytes(dtype), sms = sm_count(device);
    LinearTiles g;
    g.slices = (int)((p.k * eb + LSLICE - 1) / LSLICE);
    const ClusterRoom *room = nullptr;
    LK_TRY(cluster_room(device, &room));
    const LinearPlan plan = linear_plan(p.m, p.n, g.slices, *room);
    const int cg = plan.pair ? 2 : 1;
    g.mt = plan.mt;
    g.split = plan.split;
    g.tiles_m = (int)((p.m + g.mt - 1) / g.mt);
    g.tiles_n = (int)((p.n + LW * cg - 1) / (LW * cg));
    g.tiles = (long long)g.tiles_m * g.tiles_n;
    const long long a_bytes = p.m * p.k * eb, w_bytes = p.n * p.k * eb, keep = 48ll << 20;  // what stays in L2 beside the rest
    if (a_bytes <= w_bytes) g.band = std::min(8, g.tiles_n);
    else g.band = (int)std::min<long long>(g.tiles_n, std::max<long long>(16, keep / (LW * cg * p.k * eb)));
    g.stages = ring_stages(g.mt, cg, g.split);
    // 134 MB of w: 25.1 us with the hint, 26.4 without; 17 MB: no difference, and the next call may find it in L2
    g.w_once = g.tiles_m == 1 && p.n * p.k * eb > (64ll << 20);
    g.columns = std::max(32u, 2u * (unsigned)g.mt);
    const unsigned kinds = dtype == LK_I8 ? (2u << 4) | (1u << 7) | (1u << 10)  // int8 x int8 -> int32
                           : dtype == LK_BF16 ? (1u << 4) | (1u << 7) | (1u << 10) : (1u << 4);  // -> float32
    g.idesc = kinds | ((unsigned)(g.mt >> 3) << 17) | ((unsigned)((LW * cg) >> 4) << 24);
    CUtensorMap tw, ta;
    const long long row = p.k * eb, single = (row + 15) / 16 * 16;
    LK_TRY(encode_rows(&tw, p.w, p.n, row, p.n == 1 ? single : p.ldw * eb, LW));
    LK_TRY(encode_rows(&ta, p.a, p.m, row, p.m == 1 ? single : p.lda * eb, g.mt / cg));
    const bool i8 = dtype == LK_I8;
    if (plan.pair) return i8 ? mma_out<true, true>(tw, ta, p, g, device, sms, st) : mma_out<true, false>(tw, ta, p, g, device, sms, st);
    return i8 ? mma_out<false, true>(tw, ta, p, g, device, sms, st) : mma_out<false, false>(tw, ta, p, g, device, sms, st);
}

// Whether a wait ran out on the device since the last call; the flag is lowered.
int linear_failed(int *out) {
    unsigned v = 0, zero = 0;
    LK_CUDA(cudaMemcpyFromSymbol(&v, g_linear_failed, sizeof v));
    if (v) LK_CUDA(cudaMemcpyToSymbol(g_linear_failed, &zero, sizeof zero));
    *out = v != 0;
    return 0;
}

}  // namespace lk
