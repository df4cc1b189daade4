// e4m3 matrix product on the 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// Mathematics: gemm_f8.cuh. The f32 scales of a block of 128 cannot enter the
// tensor core, so every block's product is a fresh accumulation in TMEM (four
// kind::f8f6f4 MMAs of K = 32) that the epilogue warps read, scale and add to
// f32 registers. The activations are the MMA's M side: a thread of the
// epilogue then owns one row (one TMEM lane), its block scale is one scalar
// xs[row][b] * ws[m block][b], and the promotion is one packed FMA per two
// values.
//
// Roles of a CTA of 384 threads, one per SM, persistent over tiles of 128
// rows x BN weight rows:
//   warp 0      TMA producer: 128 x 128 bytes of x and BN x 128 bytes of w per
//               stage (128-byte swizzle); GATHER: the rows of x that a row
//               table names, four per instruction
//   warp 1      issues the MMAs of a block into one of 512 / BN TMEM buffers
//   warp 2      allocates TMEM; copies the block scales of the tile's rows and
//               weights into shared memory, transposed, in chunks of eight
//               blocks that are up to 16 blocks ahead (their first touch can
//               come from DRAM: 3500 cycles and more)
//   warp 3      gate: waits for the sums of a block and lets the epilogue warps
//               through a named barrier (a dozen warps polling shared-memory
//               barriers slow down every barrier operation: a poll of a
//               completed barrier went from 50 to 340 cycles)
//   warps 4-11  promote: two warpgroups, BN / 2 columns each; at a tile's end
//               they round, transpose through shared memory and store rows
// A block of a 128 x 256 tile is 512 cycles of MMA and 160 more until its end
// is seen, 500 to 600 of promotion (TMEM read, scale, add) and about 150 of
// hand-overs; with two TMEM buffers a block leaves every 850 to 1000 cycles.
// That bounds large products: 8192 x 4096 x 14336 bf16 497 us in a run of a few
// launches, 1.94 PFLOP/s, tensor pipe 51% busy; in a long run, where the 1000 W
// cap takes the clock down to 1.6 GHz, 580 to 596 us. Few rows are bound by the
// weights' bytes: 16 rows over experts of 4096 x 14336, five of them hit, 54 us,
// 5.4 TB/s.
//
// SPLIT: few tiles. A cluster of S CTAs shares a tile, each takes a range of
// blocks; the partial tiles meet in distributed shared memory and are added
// in rank order, so no workspace is needed and the result does not depend on
// timing. (64 rows, 4096 x 4096: 11.5 us with S = 4, 15.4 with one CTA per
// tile; the cluster itself costs 3.5 us.)
//
// Every wait for another role's progress is an mbarrier wait with a limit, so
// that a role that gives up leaves nobody behind; when one runs out the CTA
// writes NaN to its tile and to those that it has not finished, raises
// STATUS_TIMEOUT where the call has a status word, lets its copies and MMAs
// land, frees TMEM and returns.
// (TMEM buffers handed back through a named barrier, which has no limit: 32
// and 64 rows, 4096 x 14336, 0.6 to 0.9 us less of 17.2, others no different.)
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../host_common.h"
#include "gemm_f8.cuh"
#include "tc.cuh"
#include "tmap.h"

namespace fbk {

namespace {

constexpr int GM = 128;           // rows per tile
constexpr int G_EPI_WARPS = 8;
constexpr int G_EPI_GROUPS = G_EPI_WARPS / 4;
constexpr int G_THREADS = 128 + 32 * G_EPI_WARPS;
constexpr int G_XBOX = 32;        // rows per TMA box of x: only boxes with live rows are fetched
constexpr int G_MAX_E = 1024;
constexpr int G_REGS_EPI = 208, G_REGS_REST = 88;
constexpr int G_SCB = 8;          // blocks per chunk of scales
constexpr int G_SCR = 3;          // chunks in flight
constexpr int G_SCP = GM + 4;     // floats between two blocks of a chunk (the copy to it has no bank conflicts)
constexpr int G_STG = 64;         // bytes of a row that an epilogue warp stages at a time

template <int BN>
struct GCfg {
    static constexpr int X_STAGE = GM * F8B;
    static constexpr int W_STAGE = BN * F8B;
    static constexpr int STAGE = X_STAGE + W_STAGE;
    static constexpr int NS = BN == 256 ? 4 : 6;  // stages
    static constexpr int NB = 512 / BN;           // TMEM buffers
    static constexpr int COLS = BN / G_EPI_GROUPS;  // columns per epilogue warpgroup
    static constexpr int OFF_OUT = NS * STAGE;    // 32 rows of G_STG bytes per epilogue warp
    static constexpr int OFF_GRP = OFF_OUT + G_EPI_WARPS * 32 * G_STG;
    static constexpr int OFF_SX = OFF_GRP + (G_MAX_E + 1) * 4 + 12;
    static constexpr int OFF_SW = OFF_SX + G_SCR * G_SCB * G_SCP * 4;
    static constexpr int OFF_BAR = OFF_SW + G_SCR * G_SCB * 2 * 4;
    static constexpr int BYTES = OFF_BAR + (2 * NS + 2 * NB + 2 * G_SCR + 1) * 8 + 16 + 1024;
    static_assert(OFF_BAR % 8 == 0 && BYTES <= 232448, "shared memory");
    static_assert(GM * (BN + 4) * 4 <= NS * STAGE, "partial tile of a split");
};

struct GParams {
    F8Gemm p;
    int tiles_m, tiles_n;  // tiles of weight rows; of rows (ungrouped)
    int band;              // row tiles walked together (ungrouped)
    int kb;                // blocks
    int max_tiles;         // grouped: the most that groups which do not overlap can need
};

struct GTile {
    int expert, m0, row0, rows;
};

__device__ __forceinline__ void mma_f8f6f4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}

// Instruction descriptor, kind::f8f6f4: D f32, A and B e4m3, both K-major.
constexpr uint32_t f8_idesc(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

// c += a * b in c's own registers.
__device__ __forceinline__ void f2_fma_in_place(uint64_t &c, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b));
}

// The gate warp and the epilogue warps meet once per block: the kernel's only
// wait without a limit. Both sides walk every block of every tile, after an
// abort too, so they pass it in the same number.
__device__ __forceinline__ void gate_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(32 * (G_EPI_WARPS + 1)) : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Four bytes into shared memory (zero where n = 0), and the arrival of this
// thread's copies so far on a barrier.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Four rows (any four) of one 128-byte column box.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap *map, int c0, int r0, int r1, int r2, int r3,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
        : "memory");
}

// Bounded wait of a whole warp.
__device__ __forceinline__ bool tc_wait_all(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    bool ok = false;
    for (uint32_t i = 0; i < kWaitLimit; i++) {
        ok = mbar_try_wait(bar, parity);
        if (ok || ((i & 63u) == 63u && *abort_flag)) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *abort_flag = 1;
    return ok;
}

// Tile `t` (expert < 0 past the last). Ungrouped: bands of row tiles, all
// weight tiles of a band before the next band, so that the CTAs running at a
// time share both operands through L2. Grouped: `start` holds every group's
// first tile; a weight tile's row tiles are neighbours.
__device__ __forceinline__ GTile g_tile(const GParams &q, const int *start, int t, int bn) {
    if (!q.p.g.counts) {
        if (t >= q.tiles_m * q.tiles_n) return {-1, 0, 0, 0};
        const int per = q.band * q.tiles_m, b = t / per, r = t - b * per;
        const int wide = min(q.band, q.tiles_n - b * q.band);
        const int row0 = (b * q.band + r % wide) * GM;
        return {0, r / wide * bn, row0, min(GM, q.p.N - row0)};
    }
    const int E = q.p.g.n_experts;
    if (t >= start[E]) return {-1, 0, 0, 0};
    int lo = 0, hi = E;  // last group whose first tile is <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    const F8Group g = f8_group(q.p.g, lo, nullptr);
    const int nt = (g.rows + GM - 1) / GM, r = t - start[lo];
    const int at = r % nt * GM;
    return {lo, r / nt * bn, g.row0 + at, min(GM, g.rows - at)};
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float *f) {
    float v[Vec<T>::N];
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) v[i] = f[i];
    return Vec<T>::put(v);
}

// 16 bytes of one output row; element by element where the row's end or the
// alignment asks for it.
template <typename T>
__device__ __forceinline__ void store16(uint8_t *row, int m, int M, uint4 v, bool wide) {
    T *o = reinterpret_cast<T *>(row) + m;
    if (wide && m + Vec<T>::N <= M) {
        *reinterpret_cast<uint4 *>(o) = v;
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i++) {
            if (m + i >= M) break;
            if constexpr (sizeof(T) == 4)
                o[i] = __uint_as_float(w[i]);
            else
                reinterpret_cast<uint16_t *>(o)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// Columns c, c + 1, ... of a row's sums as 16 bytes of output.
template <typename T>
__device__ __forceinline__ uint4 pack_sums(const uint64_t *acc) {
    if constexpr (sizeof(T) == 4)
        return make_uint4((uint32_t)acc[0], (uint32_t)(acc[0] >> 32), (uint32_t)acc[1], (uint32_t)(acc[1] >> 32));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float x, y;
        f2_unpack(acc[sizeof(T) == 4 ? 0 : i], x, y);
        w[i] = pack2<typename std::conditional<sizeof(T) == 4, __half, T>::type>(x, y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// One warp's 32 rows x COLS columns of finished sums (a row per lane): 64
// bytes of each row at a time through 2 KB of shared memory, so that a store
// instruction covers 64 bytes of 8 rows instead of 16 bytes of 32. 16-byte
// unit u of row r lies at u ^ ((r >> 1) & 3): neither side has bank conflicts.
// `out`: the warp's first row; rows in `bad` become zeros. A whole aligned
// tile stores through four row pointers and immediate offsets: with the edge
// checks in its way the output took 15% of a tile's time (K = 4096).
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const uint64_t (&acc)[COLS / 2], uint32_t stage, uint8_t *out, uint64_t nb1, int rows,
                                           int m0, int M, uint32_t bad, int lane, bool wide) {
    constexpr int N = 16 / (int)sizeof(T);
    const int r0 = lane >> 2, u0 = lane & 3;
    const uint32_t to = stage + lane * G_STG, from = stage + r0 * G_STG + ((u0 ^ ((r0 >> 1) & 3)) << 4);
    const uint32_t sw = (lane >> 1) & 3;
    const bool whole = wide && rows >= 32 && m0 + COLS <= M && bad == 0;
    uint8_t *o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = out + (uint64_t)(i * 8 + r0) * nb1 + (uint64_t)(m0 + u0 * N) * sizeof(T);
#pragma unroll
    for (int c = 0; c < COLS; c += 4 * N) {
#pragma unroll
        for (uint32_t u = 0; u < 4; u++) sts16(to + ((u ^ sw) << 4), pack_sums<T>(&acc[(c + u * N) / 2]));
        __syncwarp();
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = lds16(from + i * 8 * G_STG);
        if (whole) {
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(o[i] + c * sizeof(T)) = v[i];
        } else {
            const int m = m0 + c + u0 * N;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (bad >> (i * 8 + r0) & 1) v[i] = make_uint4(0, 0, 0, 0);
                if (i * 8 + r0 < rows && m < M) store16<T>(out + (uint64_t)(i * 8 + r0) * nb1, m, M, v[i], wide);
            }
        }
        __syncwarp();
    }
}

template <int BN, bool SPLIT, bool GATHER, typename T>
__global__ void __launch_bounds__(G_THREADS, 1)
    gemm_f8_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                   const __grid_constant__ GParams q) {
    using C = GCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (sbase - smem_u32(smem_raw));
    int *start = reinterpret_cast<int *>(gbase + C::OFF_GRP);
    uint64_t *full = reinterpret_cast<uint64_t *>(gbase + C::OFF_BAR);
    uint64_t *empty = full + C::NS;
    uint64_t *t_full = empty + C::NS;
    uint64_t *t_empty = t_full + C::NB;
    uint64_t *s_full = t_empty + C::NB;
    uint64_t *s_empty = s_full + G_SCR;
    uint64_t *drained = s_empty + G_SCR;
    float *sx = reinterpret_cast<float *>(gbase + C::OFF_SX);
    float *sw = reinterpret_cast<float *>(gbase + C::OFF_SW);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const F8Gemm &p = q.p;

    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_x) : "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < C::NS; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < C::NB; i++) {
            mbar_init(&t_full[i], 1);
            mbar_init(&t_empty[i], G_EPI_WARPS);
        }
        for (int i = 0; i < G_SCR; i++) {
            mbar_init(&s_full[i], 32);
            mbar_init(&s_empty[i], G_EPI_WARPS);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // (up to here no global memory: the set-up overlaps the end of the stream's previous kernel)
    grid_dependency_wait();
    grid_launch_dependents();
    if (warp == 3 && p.g.counts) {  // first tile of every group
        // (overlapping groups could ask for any number of tiles: no more than
        // max_tiles are walked)
        int run = 0;
        bool over = false;
        for (int e0 = 0; e0 < p.g.n_experts; e0 += 32) {
            int n = 0;
            if (e0 + lane < p.g.n_experts)
                n = (f8_group(p.g, e0 + lane, blockIdx.x == 0 ? p.status : nullptr).rows + GM - 1) / GM * q.tiles_m;
            int64_t sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            if (e0 + lane < p.g.n_experts) start[e0 + lane] = (int)min(run + sum - n, (int64_t)q.max_tiles);
            const int64_t all = run + __shfl_sync(0xffffffffu, sum, 31);
            over = over || all > q.max_tiles;
            run = (int)min(all, (int64_t)q.max_tiles);
        }
        if (lane == 0) {
            start[p.g.n_experts] = run;
            if (over && blockIdx.x == 0) report_status(p.status, STATUS_BAD_ID);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int S = SPLIT ? (int)cluster_size() : 1, rank = SPLIT ? (int)cluster_rank() : 0;
    const int t0 = (int)blockIdx.x / S, t_step = SPLIT ? 0x40000000 : (int)gridDim.x;
    const int b0 = SPLIT ? (int)((int64_t)q.kb * rank / S) : 0, b1 = SPLIT ? (int)((int64_t)q.kb * (rank + 1) / S) : q.kb;

    int copied = 0;  // producer: stages that copies were issued for
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G_REGS_REST));
        if (warp == 0) {
            // ---- TMA producer ---------------------------------------------------
            int it = 0;
            bool ok = true;
            for (int t = t0; ok; t += t_step) {
                const GTile tile = g_tile(q, start, t, BN);
                if (tile.expert < 0) break;
                int r[4] = {0, 0, 0, 0};
                if constexpr (GATHER) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (lane * 4 + j < tile.rows) r[j] = max(0, f8_source(p.g, tile.row0 + lane * 4 + j, nullptr));
                }
                const int boxes = (tile.rows + (GATHER ? 3 : G_XBOX - 1)) / (GATHER ? 4 : G_XBOX);
                const uint32_t bytes = C::W_STAGE + boxes * (GATHER ? 4 : G_XBOX) * F8B;
                for (int b = b0; b < b1; b++, it++) {
                    const int s = it % C::NS;
                    if (!tc_wait_warp(&empty[s], ((it / C::NS) & 1) ^ 1, abort_flag, lane, 20)) {
                        ok = false;
                        break;
                    }
                    const uint32_t xs = sbase + s * C::STAGE, ws = xs + C::X_STAGE, bar = smem_u32(&full[s]);
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&full[s], bytes);
                        tma_load_3d(ws, &tm_w, b * F8B, tile.m0, tile.expert, bar);
                    }
                    __syncwarp();
                    if (GATHER) {
                        if (lane < boxes) tma_gather4(xs + lane * 4 * F8B, &tm_x, b * F8B, r[0], r[1], r[2], r[3], bar);
                    } else if (lane < boxes) {
                        tma_load_2d(xs + lane * G_XBOX * F8B, &tm_x, b * F8B, tile.row0 + lane * G_XBOX, bar);
                    }
                }
            }
            copied = it;
        } else if (warp == 1) {
            // ---- MMA issuer -----------------------------------------------------
            // (the whole warp walks the loop and one elected lane issues: with
            // warp-uniform operands an MMA issues in a few cycles, from a
            // divergent branch in about 50)
            constexpr uint32_t idesc = f8_idesc(GM, BN);
            const uint64_t desc0 = sw128_desc(sbase);
            int it = 0;
            bool ok = true;
            for (int t = t0;; t += t_step) {
                if (g_tile(q, start, t, BN).expert < 0) break;
                for (int b = b0; b < b1; b++, it++) {
                    const int s = it % C::NS, u = it % C::NB;
                    ok = ok && tc_wait_all(&full[s], (it / C::NS) & 1, abort_flag) &&
                         tc_wait_all(&t_empty[u], ((it / C::NB) & 1) ^ 1, abort_flag);
                    if (!ok) continue;
                    tc_fence_after();
                    const uint64_t xd = desc0 + (uint64_t)(s * (C::STAGE / 16)), wd = xd + C::X_STAGE / 16;
                    const uint32_t d = tmem + (uint32_t)(u * BN);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < F8B / 32; k++) mma_f8f6f4(d, xd + k * 2, wd + k * 2, idesc, k ? 1u : 0u);
                        tc_commit(smem_u32(&t_full[u]));
                        tc_commit(smem_u32(&empty[s]));
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) tc_commit(smem_u32(drained));  // every MMA issued here
        } else if (warp == 2) {
            // ---- scales: G_SCB blocks of 128 rows at a time, eight lanes per row -------------
            const int j = lane & 7;
            int ch = 0;
            bool ok = true;
            for (int t = t0; ok; t += t_step) {
                const GTile tile = g_tile(q, start, t, BN);
                if (tile.expert < 0) break;
                int src[4];  // scale rows of tile rows lane, 32 + lane, ...
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = i * 32 + lane;
                    src[i] = -1;
                    if (r < tile.rows) src[i] = p.g.counts ? f8_source(p.g, tile.row0 + r, nullptr) : tile.row0 + r;
                }
                const int mb = tile.m0 / F8B + (lane >> 3), mbs = (p.M + F8B - 1) / F8B;
                const uint8_t *wr = p.ws + (uint64_t)tile.expert * p.ws_nb2 + (uint64_t)min(mb, mbs - 1) * p.ws_nb1;
                for (int b = b0; b < b1; b += G_SCB, ch++) {
                    const int c = ch % G_SCR;
                    if (!tc_wait_warp(&s_empty[c], ((ch / G_SCR) & 1) ^ 1, abort_flag, lane, 100)) {
                        ok = false;
                        break;
                    }
                    const bool in = b + j < b1;
                    if (lane < 16 && in) cp_async4(smem_u32(&sw[(c * G_SCB + j) * 2 + (lane >> 3)]), wr + (b + j) * 4, 4);
                    const uint32_t dst = smem_u32(&sx[(c * G_SCB + j) * G_SCP + (lane >> 3)]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const int r = __shfl_sync(0xffffffffu, src[i], e * 4 + (lane >> 3));
                            const bool get = r >= 0 && in;
                            cp_async4(dst + (i * 32 + e * 4) * 4, p.xs + (get ? (uint64_t)r * p.xs_nb1 + (b + j) * 4 : 0), get ? 4 : 0);
                        }
                    }
                    cp_async_arrive(&s_full[c]);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            // ---- gate: waits for a block's sums (and scales) on the epilogue's behalf --------------
            // (after an abort it lets every remaining step through without waiting)
            int it = 0, ch = 0;
            bool ok = true;
            for (int t = t0;; t += t_step) {
                if (g_tile(q, start, t, BN).expert < 0) break;
                for (int b = b0; b < b1; b++, it++) {
                    const int u = it % C::NB;
                    if ((b - b0) % G_SCB == 0) {
                        ok = ok && tc_wait_all(&s_full[ch % G_SCR], (ch / G_SCR) & 1, abort_flag);
                        ch++;
                    }
                    ok = ok && tc_wait_all(&t_full[u], (it / C::NB) & 1, abort_flag);
                    gate_sync();
                }
            }
        }
    } else {
        // ---- promotion and output -------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G_REGS_EPI));
        const int ew = warp - 4, part = ew & 3, grp = ew >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(part * 32) << 16) + (uint32_t)(grp * C::COLS);
        const uint32_t stage = sbase + C::OFF_OUT + ew * 32 * G_STG;
        int it = 0, ch = 0;
        for (int t = t0;; t += t_step) {
            if (g_tile(q, start, t, BN).expert < 0) break;
            const int r_first = part * 32, row = r_first + lane;
            uint64_t acc[C::COLS / 2];
#pragma unroll
            for (int i = 0; i < C::COLS / 2; i++) acc[i] = 0;
            float sc = 0.0f;
#pragma unroll 1
            for (int b = b0; b < b1; b++, it++) {
                const int u = it % C::NB, j = (b - b0) % G_SCB, c = ch % G_SCR;
                gate_sync();
                // a warpgroup's columns lie in one block row of the weights; the
                // scales of the next block are read behind this block's loads
                const float *sxc = &sx[c * G_SCB * G_SCP + row], *swc = &sw[c * G_SCB * 2 + grp * C::COLS / F8B];
                if (j == 0) sc = sxc[0] * swc[0];
                tc_fence_after();
                const uint64_t sc2 = f2_pack(sc, sc);
                uint32_t v[2][16];
                tc_ld16(lanes + (uint32_t)(u * BN), v[0]);
                const int jn = j + 1 < G_SCB ? j + 1 : 0;
                sc = sxc[jn * G_SCP] * swc[jn * 2];
                tc_wait_ld();
#pragma unroll
                for (int h = 0; h < C::COLS / 16; h++) {
                    if (h + 1 < C::COLS / 16) tc_ld16(lanes + (uint32_t)(u * BN + (h + 1) * 16), v[(h + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        f2_fma_in_place(acc[h * 8 + i], f2_pack_bits(v[h & 1][2 * i], v[h & 1][2 * i + 1]), sc2);
                    if (h + 1 < C::COLS / 16) tc_wait_ld();
                    if (h + 2 == C::COLS / 16) {  // all of it is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&t_empty[u]);
                    }
                }
                if (j == G_SCB - 1 || b == b1 - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_empty[c]);
                    ch++;
                }
            }
            // (the tile again: kept across the loop it costs the accumulators' registers)
            int t2 = t;
            asm volatile("" : "+r"(t2));
            const GTile tile = g_tile(q, start, t2, BN);
            int src = -1;
            if (row < tile.rows) src = p.g.counts ? f8_origin(p.g, tile.row0 + row, p.status) : 0;
            if constexpr (SPLIT) {
                // the pipeline's stages are free: every copy was consumed and every MMA has been read
                float *mine = reinterpret_cast<float *>(gbase) + row * (BN + 4) + grp * C::COLS;
                if (row < tile.rows) {
#pragma unroll
                    for (int i = 0; i < C::COLS / 2; i += 2)
                        *reinterpret_cast<ulonglong2 *>(mine + 2 * i) = make_ulonglong2(src >= 0 ? acc[i] : 0, src >= 0 ? acc[i + 1] : 0);
                }
            } else {
                const uint32_t bad = __ballot_sync(0xffffffffu, src < 0);
                const bool wide = ((reinterpret_cast<uintptr_t>(p.y) | p.y_nb1) & 15) == 0;
                const int rows = tile.rows - r_first;
                // (set before the gate lets the first block through that is not
                // what it should be: where it is still clear the sums are right)
                if (*abort_flag) {
#pragma unroll
                    for (int i = 0; i < C::COLS / 2; i++) acc[i] = 0x7fffffff7fffffffull;
                }
                if (rows > 0)
                    store_rows<T, C::COLS>(acc, stage, p.y + (uint64_t)(tile.row0 + r_first) * p.y_nb1, p.y_nb1, rows,
                                           tile.m0 + grp * C::COLS, p.M, bad, lane, wide);
            }
        }
    }
    __syncthreads();
    // whoever aborted, and whenever: no copy outlives the CTA
    if (warp == 0 && *abort_flag)
        for (int i = max(0, copied - C::NS); i < copied; i++) mbar_wait_bounded(&full[i % C::NS], (i / C::NS) & 1);
    __syncwarp();
    if constexpr (SPLIT) {
        cluster_arrive();
        cluster_wait();
        const GTile tile = g_tile(q, start, t0, BN);
        int broken = 0;  // in any CTA of the cluster
        for (int i = 0; i < S; i++) broken |= (int)dsmem_ld4(dsmem_map(const_cast<const int *>(abort_flag), (uint32_t)i));
        static_assert(!SPLIT || BN == 128, "four columns per lane");
        if (tile.expert >= 0) {
            // rows rank, rank + S, ...: the S partial rows, all of them on the way
            // before the first is added (one after the other they cost 3 us),
            // in rank order
            const int m = tile.m0 + lane * 4;
            const bool wide = ((reinterpret_cast<uintptr_t>(p.y) | p.y_nb1) & (4 * sizeof(T) - 1)) == 0 && m + 4 <= p.M;
            for (int r = rank + warp * S; r < tile.rows; r += G_THREADS / 32 * S) {
                const uint8_t *mine = gbase + (r * (BN + 4) + lane * 4) * 4;
                int4 v[8];
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < S) v[i] = dsmem_ld16(dsmem_map(mine, (uint32_t)i));
                float f[4] = {};
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < S) {
                        f[0] += __int_as_float(v[i].x);
                        f[1] += __int_as_float(v[i].y);
                        f[2] += __int_as_float(v[i].z);
                        f[3] += __int_as_float(v[i].w);
                    }
                if (broken) f[0] = f[1] = f[2] = f[3] = __int_as_float(0x7fffffff);
                T *o = reinterpret_cast<T *>(p.y + (uint64_t)(tile.row0 + r) * p.y_nb1) + m;
                if (wide) {
                    if constexpr (sizeof(T) == 4)
                        *reinterpret_cast<float4 *>(o) = make_float4(f[0], f[1], f[2], f[3]);
                    else
                        *reinterpret_cast<uint2 *>(o) = make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (m + i < p.M) o[i] = from_f32<T>(f[i]);
                }
            }
        }
        cluster_arrive();
        cluster_wait();
    }
    if (*abort_flag && tid == 0) report_status(p.status, STATUS_TIMEOUT);
    if (warp == 2) {
        mbar_wait_bounded(drained, 0);
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Gathered copies: a warp per row. A row whose table entry is out of range is
// left as it is: the product checks the table again and writes zeros.
__global__ void __launch_bounds__(256) gather_f8_kernel(const F8Gemm p, uint8_t *xg, uint64_t xg_nb1, float *sg, int kb) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= p.g.n_rows) return;
    const int src = f8_source(p.g, r, nullptr);
    if (src < 0) return;
    const uint8_t *x = p.x + (uint64_t)src * p.x_nb1;
    uint8_t *o = xg + (uint64_t)r * xg_nb1;
    for (int k = lane * 16; k < p.K; k += 512) {
        if (k + 16 <= p.K)
            *reinterpret_cast<uint4 *>(o + k) = ld_stream16(x + k);
        else
            for (int i = k; i < p.K; i++) o[i] = x[i];
    }
    const float *s = reinterpret_cast<const float *>(p.xs + (uint64_t)src * p.xs_nb1);
    for (int b = lane; b < kb; b += 32) sg[(int64_t)r * kb + b] = s[b];
}

template <int BN, bool SPLIT, bool GATHER, typename T>
int launch_t(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const GParams &q, int ctas, int cluster, cudaStream_t s) {
    using C = GCfg<BN>;
    auto *fn = gemm_f8_kernel<BN, SPLIT, GATHER, T>;
    static DeviceFlags done;
    int rc = raise_smem_limit(reinterpret_cast<const void *>(fn), C::BYTES, done, "mul_mat_f8");
    if (rc) return rc;
    // setmaxnreg draws on the registers of the launch: the two shares must fit
    static const int regs = [] {
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, reinterpret_cast<const void *>(gemm_f8_kernel<BN, SPLIT, GATHER, T>)) == cudaSuccess ? a.numRegs : 0;
    }();
    if (regs * G_THREADS < 32 * G_EPI_WARPS * G_REGS_EPI + 128 * G_REGS_REST)
        return fb::set_error(FB_ERR_CUDA, "mul_mat_f8: built with %d registers per thread", regs);
    return launch_early("mul_mat_f8", gemm_f8_kernel<BN, SPLIT, GATHER, T>, dim3((unsigned)ctas), dim3(G_THREADS), C::BYTES, cluster, s,
                        tm_w, tm_x, q);
}

template <int BN, bool SPLIT, bool GATHER>
int launch_o(const CUtensorMap &tm_w, const CUtensorMap &tm_x, const GParams &q, int ctas, int cluster, cudaStream_t s) {
    if (q.p.out_type == FB_F32) return launch_t<BN, SPLIT, GATHER, float>(tm_w, tm_x, q, ctas, cluster, s);
    if (q.p.out_type == FB_F16) return launch_t<BN, SPLIT, GATHER, __half>(tm_w, tm_x, q, ctas, cluster, s);
    return launch_t<BN, SPLIT, GATHER, __nv_bfloat16>(tm_w, tm_x, q, ctas, cluster, s);
}

template <int BN, bool SPLIT>
int launch_g(bool gather, const CUtensorMap &tm_w, const CUtensorMap &tm_x, const GParams &q, int ctas, int cluster,
             cudaStream_t s) {
    return gather ? launch_o<BN, SPLIT, true>(tm_w, tm_x, q, ctas, cluster, s)
                  : launch_o<BN, SPLIT, false>(tm_w, tm_x, q, ctas, cluster, s);
}

}  // namespace

bool gemm_f8_supported(const F8Gemm &p) {
    auto ok = [](const void *a, uint64_t nb) { return ((reinterpret_cast<uintptr_t>(a) | nb) & 15) == 0 && nb < (1ull << 40); };
    if (!ok(p.w, p.w_nb1) || !ok(p.x, p.x_nb1)) return false;
    // planes of experts, one behind the other
    return p.g.n_experts <= 1 || (p.w_nb2 % 16 == 0 && p.w_nb2 < (1ull << 40) && p.w_nb2 >= (uint64_t)p.M * p.w_nb1);
}

uint64_t gather_f8_bytes(int64_t K, int64_t n_rows) {
    return (uint64_t)n_rows * (uint64_t)((K + 15) / 16 * 16) + (uint64_t)n_rows * (uint64_t)((K + F8B - 1) / F8B * 4);
}

// TMA gathers four rows per instruction and about 90 cycles, beside a block's
// weights that take 1400 cycles of memory bandwidth: up to 16 rows per tile
// it is free, at 128 rows it doubled the time of the product (8 experts x
// [4096, 14336], 1024 rows: 242 us, with the gathered copy 121 us).
bool gather_f8_pays(int64_t n_rows, int64_t n_experts) { return n_rows > 16 * n_experts; }

int launch_gather_f8(F8Gemm &p, void *ws, cudaStream_t s) {
    const uint64_t nb1 = (uint64_t)(p.K + 15) / 16 * 16;
    uint8_t *xg = static_cast<uint8_t *>(ws);
    float *sg = reinterpret_cast<float *>(xg + (uint64_t)p.g.n_rows * nb1);
    const int kb = (p.K + F8B - 1) / F8B;
    const int rc = launch_early("mul_mat_f8_grouped", gather_f8_kernel, dim3((unsigned)(((int64_t)p.g.n_rows + 7) / 8)), dim3(256), 0, 1,
                                s, p, xg, nb1, sg, kb);
    if (rc) return rc;
    p.x = xg;
    p.x_nb1 = nb1;
    p.xs = reinterpret_cast<const uint8_t *>(sg);
    p.xs_nb1 = (uint64_t)kb * 4;
    p.g.gathered = p.g.rows;
    p.g.n_origin = p.g.n_x;
    p.g.rows = nullptr;
    p.g.n_x = p.g.n_rows;
    return FB_OK;
}

F8Plan gemm_f8_plan(int64_t K, int64_t M, int64_t N, int64_t n_experts) {
    const int sms = sm_count();
    const int64_t kb = (K + F8B - 1) / F8B, m128 = (M + 127) / 128, m256 = (M + 255) / 256;
    // row tiles: exact, or the most that the groups can need
    const int64_t nt = n_experts ? std::min<int64_t>(N, N / GM + std::min<int64_t>(n_experts, N)) : (N + GM - 1) / GM;
    // A block of a 128-column tile takes about 2/3 of the time of a 256-column
    // one, so the wider tile wins unless the narrower saves a third of the
    // rounds over the SMs or can be split (1024 rows, 4096 x 4096: 22.7 us at
    // 256 columns, 33.7 at 128; 64 rows, 4096 x 14336: 21.4 and 17.4; 256 rows,
    // 4096 x 4096: 20.9 and, in two, 15.4). Grouped products follow the same
    // rule from the most tiles that their groups can need (8 experts of 4096 x
    // 14336, 16 rows: 54.9 us at 256 columns, 64.0 at 128; 1024 rows: 121.8,
    // 165.0; 64 of 1408 x 2048, 18006 rows: 104, 128), though with few experts
    // hit the narrower tile can be a little faster (two tokens: 51.6, 50.3).
    const int64_t cost256 = 3 * ((nt * m256 + sms - 1) / sms), cost128 = 2 * ((nt * m128 + sms - 1) / sms);
    F8Plan f{};
    f.tile = cost256 <= cost128 ? 256 : 128;
    f.warps = G_THREADS / 32;
    f.row_tiles = nt;
    f.tiles = nt * (f.tile == 256 ? m256 : m128);
    f.split = 1;
    if (f.tile == 128)
        while (f.split < 8 && f.tiles * f.split * 2 <= sms && kb / (f.split * 2) >= 2) f.split *= 2;
    // a block is 0.37 us, a cluster 3.5 us (64 rows, 1024 x 1024: 6.4 us in one, 7.9 in four)
    if (kb * (f.split - 1) < 12 * f.split) f.split = 1;
    f.ctas = f.split > 1 ? f.tiles * f.split : std::min<int64_t>(f.tiles, sms);
    return f;
}

int launch_gemm_f8(const F8Gemm &p, cudaStream_t s) {
    const bool grouped = p.g.counts != nullptr, gather = grouped && p.g.rows;
    const int64_t n_exp = grouped ? p.g.n_experts : 1;
    const F8Plan f = gemm_f8_plan(p.K, p.M, p.N, grouped ? n_exp : 0);
    if (f.row_tiles * ((p.M + 127) / 128) > INT32_MAX / 2) return fb::set_error(FB_ERR_UNSUPPORTED, "mul_mat_f8: too many tiles");
    const int bn = f.tile, split = f.split, ctas = (int)f.ctas;
    GParams q{};
    q.p = p;
    q.kb = (p.K + F8B - 1) / F8B;
    q.tiles_n = (int)f.row_tiles;
    // (16: 2048 rows, 4096 x 14336 129.9 us, 8192 rows 498; row tiles one by one
    // 140.9 and 519; eight 131.6 and 504; 64 130.2 and 497, but 4096 rows of 4096 x
    // 4096 81.7 instead of 77.6)
    q.band = 16;
    q.tiles_m = (p.M + bn - 1) / bn;
    q.max_tiles = (int)f.tiles;
    CUtensorMap tm_w, tm_x;
    int rc = encode_tensor_map_3d_sw128(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.w, (uint64_t)p.K, (uint64_t)p.M,
                                        (uint64_t)n_exp, p.w_nb1, n_exp > 1 ? p.w_nb2 : p.w_nb1 * (uint64_t)p.M, F8B,
                                        (uint32_t)bn);
    if (rc) return rc;
    rc = encode_tensor_map_2d_sw128(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.x, (uint64_t)p.K,
                                    (uint64_t)(grouped ? p.g.n_x : p.N), p.x_nb1, F8B, gather ? 1 : G_XBOX);
    if (rc) return rc;
    if (split > 1) return launch_g<128, true>(gather, tm_w, tm_x, q, ctas, split, s);
    if (bn == 256) return launch_g<256, false>(gather, tm_w, tm_x, q, ctas, 1, s);
    return launch_g<128, false>(gather, tm_w, tm_x, q, ctas, 1, s);
}

}  // namespace fbk
