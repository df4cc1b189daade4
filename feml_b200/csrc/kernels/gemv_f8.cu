// e4m3 matrix product for few rows of x (a decode step): the weights are read
// once, straight into tensor-core fragments.
//
// A warp takes 32 weight rows x one block of 128 values at a time: thread
// (g, t) of the m16n8k16 layout loads bytes 32 t to 32 t + 31 of rows g, g + 8,
// g + 16 and g + 24. The layout's own order of k within a row does not matter
// to a sum as long as both operands use the same one, so a 32-bit word of each
// row serves one MMA and nothing is shuffled. The words are widened to f16 on
// the way (exact; the sum is f32): the MMA that takes e4m3 itself measured
// about 100 cycles per instruction here, several times the conversions and
// f16 MMAs that replace it. The products of a block are scaled in registers;
// the warps of a CTA take blocks in turn and meet in shared memory in warp
// order. Few weight rows: a cluster of S CTAs splits the blocks further and
// adds its partial sums in rank order through distributed shared memory.
// Bound by memory: each warp has two blocks (8 KB of weights) in flight (one
// row, 4096 x 4096: 5.3 us, 3.2 TB/s; 4096 x 14336: 13.9 us, 4.2 TB/s; launch
// and one memory round trip are 3 us of either). Two groups of eight rows at
// sixteen warps do not fit 128 registers: 92 bytes spilled with 16-byte loads,
// 156 with 32-byte ones (16 rows, 4096 x 4096: 7.0 us).
#include <cuda_runtime.h>

#include <algorithm>

#include "../host_common.h"
#include "gemm_f8.cuh"

namespace fbk {

namespace {

constexpr int V_TILES = 2;   // m16 tiles of weight rows per warp
constexpr int V_ROWS = 16 * V_TILES;

// The 16-byte unit at `p`, of which `n` bytes exist (the end of a row).
__device__ __forceinline__ uint4 ld_unit(const uint8_t *p, int n) {
    if (n >= 16) return ld_stream16(p);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < n; i++) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four e4m3 values as two pairs of f16.
__device__ __forceinline__ void widen(uint32_t v, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(v));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of eight rows of x. WIDE: weight rows aligned to 32 bytes.
// V_WARPS: warps that take blocks in turn.
template <int V_WARPS, int NT, bool WIDE, typename T>
__global__ void __launch_bounds__(32 * V_WARPS, V_WARPS == 8 && NT == 1 ? 2 : 1) gemv_f8_kernel(const F8Gemm p, int splits) {
    __shared__ float part[V_WARPS][NT * 8][V_ROWS + 1];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = (int)(blockIdx.x / splits) * V_ROWS, rank = (int)(blockIdx.x % splits);
    const int kb = (p.K + F8B - 1) / F8B;
    const uint8_t *w[2 * V_TILES];
#pragma unroll
    for (int i = 0; i < 2 * V_TILES; i++) w[i] = p.w + (uint64_t)min(m0 + g + 8 * i, p.M - 1) * p.w_nb1 + t * 32;
    const uint8_t *x[NT];
    const float *xs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        x[n] = p.x + (uint64_t)min(n * 8 + g, p.N - 1) * p.x_nb1 + t * 32;
#pragma unroll
        for (int h = 0; h < 2; h++)
            xs[n][h] = reinterpret_cast<const float *>(p.xs + (uint64_t)min(n * 8 + 2 * t + h, p.N - 1) * p.xs_nb1);
    }
    // (32 weight rows lie in one block row)
    const float *ws = reinterpret_cast<const float *>(p.ws + (uint64_t)(m0 / F8B) * p.ws_nb1);
    float acc[NT][V_TILES][4] = {};
    auto product = [&](const uint4 (&a)[2 * V_TILES][2], const uint4 (&xv)[NT][2], const float (&s)[NT][2]) {
        float d[NT][V_TILES][4] = {};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                auto word = [&](const uint4 &v) { return c == 0 ? v.x : c == 1 ? v.y : c == 2 ? v.z : v.w; };
                uint32_t b[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++) widen(word(xv[n][h]), b[n][0], b[n][1]);
#pragma unroll
                for (int i = 0; i < V_TILES; i++) {
                    uint32_t a0, a1, a2, a3;
                    widen(word(a[2 * i][h]), a0, a2);
                    widen(word(a[2 * i + 1][h]), a1, a3);
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_f16(d[n][i], a0, a1, a2, a3, b[n][0], b[n][1]);
                }
            }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < V_TILES; i++)
#pragma unroll
                for (int h = 0; h < 4; h++) acc[n][i][h] = fmaf(d[n][i][h], s[n][h & 1], acc[n][i][h]);
    };
    const int whole = p.K / F8B, step = V_WARPS * splits;
    auto fetch = [&](int b, uint4 (&a)[2 * V_TILES][2]) {
#pragma unroll
        for (int r = 0; r < 2 * V_TILES; r++) {
            const uint8_t *q = w[r] + (int64_t)b * F8B;
            if constexpr (WIDE) {
                const Wide32 v = ld_stream32(q);
                a[r][0] = v.lo;
                a[r][1] = v.hi;
            } else {
                a[r][0] = ld_stream16(q);
                a[r][1] = ld_stream16(q + 16);
            }
        }
    };
    auto use = [&](int b, const uint4 (&a)[2 * V_TILES][2]) {
        uint4 xv[NT][2];
        float s[NT][2];
        const float sw = ws[b];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            xv[n][0] = *reinterpret_cast<const uint4 *>(x[n] + (int64_t)b * F8B);
            xv[n][1] = *reinterpret_cast<const uint4 *>(x[n] + (int64_t)b * F8B + 16);
            s[n][0] = xs[n][0][b] * sw;
            s[n][1] = xs[n][1][b] * sw;
        }
        product(a, xv, s);
    };
    int b = rank * V_WARPS + warp;
    for (; b < whole; b += 2 * step) {
        uint4 a0[2 * V_TILES][2], a1[2 * V_TILES][2];
        fetch(b, a0);
        if (b + step < whole) fetch(b + step, a1);
        use(b, a0);
        if (b + step < whole) use(b + step, a1);
    }
    if (whole < kb && whole % step == rank * V_WARPS + warp) {  // the row's last, shorter block
        uint4 a[2 * V_TILES][2], xv[NT][2];
        float s[NT][2];
        const int k = whole * F8B, left = p.K - k - t * 32;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int n1 = left - 16 * h;
#pragma unroll
            for (int r = 0; r < 2 * V_TILES; r++) a[r][h] = ld_unit(w[r] + k + 16 * h, n1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                xv[n][h] = ld_unit(x[n] + k + 16 * h, n1);
                s[n][h] = xs[n][h][whole] * ws[whole];
            }
        }
        product(a, xv, s);
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < V_TILES; i++)
#pragma unroll
            for (int h = 0; h < 4; h++) part[warp][n * 8 + 2 * t + (h & 1)][i * 16 + g + (h >> 1) * 8] = acc[n][i][h];
    __syncthreads();
    constexpr int OUT = NT * 8 * V_ROWS;
    if (splits > 1) {
        for (int i = threadIdx.x; i < OUT; i += 32 * V_WARPS) {
            const int n = i / V_ROWS, r = i % V_ROWS;
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < V_WARPS; j++) v += part[j][n][r];
            part[0][n][r] = v;  // (read and written by this thread alone)
        }
        cluster_arrive();
        cluster_wait();
    }
    for (int i = threadIdx.x + rank * 32 * V_WARPS; i < OUT; i += 32 * V_WARPS * splits) {
        const int n = i / V_ROWS, r = i % V_ROWS;
        float v = 0.0f;
        if (splits > 1) {
            for (int j = 0; j < splits; j++) v += __uint_as_float(dsmem_ld4(dsmem_map(&part[0][n][r], (uint32_t)j)));
        } else {
#pragma unroll
            for (int j = 0; j < V_WARPS; j++) v += part[j][n][r];
        }
        if (n < p.N && m0 + r < p.M) reinterpret_cast<T *>(p.y + (uint64_t)n * p.y_nb1)[m0 + r] = from_f32<T>(v);
    }
    if (splits > 1) {  // a CTA's shared memory outlives its readers
        cluster_arrive();
        cluster_wait();
    }
}

template <int V_WARPS, int NT, bool WIDE, typename T>
int launch_v(const F8Gemm &p, int ctas, int splits, cudaStream_t s) {
    return launch_early("mul_mat_f8", gemv_f8_kernel<V_WARPS, NT, WIDE, T>, dim3((unsigned)ctas), dim3(32 * V_WARPS), 0, splits, s, p, splits);
}

template <int V_WARPS, typename T>
int launch_n(const F8Gemm &p, int ctas, int splits, cudaStream_t s) {
    const bool wide = ((reinterpret_cast<uintptr_t>(p.w) | p.w_nb1) & 31) == 0;
    if (p.N <= 8) return wide ? launch_v<V_WARPS, 1, true, T>(p, ctas, splits, s) : launch_v<V_WARPS, 1, false, T>(p, ctas, splits, s);
    return wide ? launch_v<V_WARPS, 2, true, T>(p, ctas, splits, s) : launch_v<V_WARPS, 2, false, T>(p, ctas, splits, s);
}

template <typename T>
int launch_w(const F8Gemm &p, int warps, int ctas, int splits, cudaStream_t s) {
    return warps == 16 ? launch_n<16, T>(p, ctas, splits, s) : launch_n<8, T>(p, ctas, splits, s);
}

}  // namespace

int gemv_f8_max_rows() { return 16; }

F8Plan gemv_f8_plan(int64_t K, int64_t M) {
    const int64_t tiles = (M + V_ROWS - 1) / V_ROWS, kb = (K + F8B - 1) / F8B;
    // Two CTAs of eight warps per SM where there are tiles enough; one of
    // sixteen where there are not and every warp has a block (one row, 4096 x
    // 4096: 5.3 us, with eight warps 6.7, with clusters of two 8.7; 2048 x 4096:
    // 3.8 and 4.3; below 16 blocks, 1024 x 4096 with 16 rows, eight take 3.4 and
    // sixteen 4.1; not borne out at 2048 x 8192, 6.8 and with eight 5.5, and at
    // 16 rows of 2048 x 4096, 5.4 and 4.3); clusters of eight-warp CTAs only where
    // the tiles do not reach half of the SMs (16384 x 512: 5.4 us with eight CTAs
    // per tile, 17 with one) and every warp keeps two blocks or more (16 rows,
    // 8192 x 512: 4.8 us, down to one block each 7.8; one row of 4096 x 512 would
    // gain: 3.9 and 3.2).
    const bool few = tiles * 2 <= sm_count();
    F8Plan f{};
    f.tile = V_ROWS;
    f.warps = few || tiles >= 2 * sm_count() || kb < 16 ? 8 : 16;
    f.row_tiles = 1;
    f.tiles = tiles;
    f.split = 1;
    while (few && f.split < 8 && tiles * f.split * 2 <= sm_count() && kb >= 4 * f.split * f.warps) f.split *= 2;
    f.ctas = tiles * f.split;
    return f;
}

int launch_gemv_f8(const F8Gemm &p, cudaStream_t s) {
    const F8Plan f = gemv_f8_plan(p.K, p.M);
    if (f.ctas > INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, "mul_mat_f8: too many tiles");
    const int warps = f.warps, ctas = (int)f.ctas, splits = f.split;
    if (p.out_type == FB_F32) return launch_w<float>(p, warps, ctas, splits, s);
    if (p.out_type == FB_F16) return launch_w<__half>(p, warps, ctas, splits, s);
    return launch_w<__nv_bfloat16>(p, warps, ctas, splits, s);
}

}  // namespace fbk
