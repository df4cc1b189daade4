// e4m3 matrix product for few rows of x (a decode step): the weights are read
// once, straight into tensor-core fragments.
//
// A warp takes 32 weight rows x one block of 128 values at a time: thread
// (g, t) of the m16n8k16 layout loads the 16-byte units t and t + 4 of rows
// g, g + 8, g + 16 and g + 24. The layout's own order of k within a row does
// not matter to a sum as long as both operands use the same one, so a 32-bit
// word of each row serves one MMA and nothing is shuffled. The words are
// widened to f16 on the way (exact; the sum is f32): the MMA that takes e4m3
// itself measured about 100 cycles per instruction here, several times the
// conversions and f16 MMAs that replace it. The products of a block are
// scaled in registers; the eight warps of a CTA take blocks in turn and meet
// in shared memory in warp order. Few weight rows: a cluster of S CTAs splits
// the blocks further and adds its partial sums in rank order through
// distributed shared memory. Bound by memory: each warp has two blocks (8 KB
// of weights) in flight.
#include <cuda_runtime.h>

#include <algorithm>

#include "../host_common.h"
#include "gemm_f8.cuh"

namespace fbk {

namespace {

constexpr int V_WARPS = 8;
constexpr int V_TILES = 2;   // m16 tiles of weight rows per warp
constexpr int V_ROWS = 16 * V_TILES;
constexpr int V_AHEAD = 2;   // blocks (4 KB each) in flight per warp

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

// NT: groups of eight rows of x.
template <int NT, typename T>
__global__ void __launch_bounds__(32 * V_WARPS) gemv_f8_kernel(const F8Gemm p, int splits) {
    __shared__ float part[V_WARPS][NT * 8][V_ROWS + 1];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = (int)(blockIdx.x / splits) * V_ROWS, rank = (int)(blockIdx.x % splits);
    const int kb = (p.K + F8B - 1) / F8B;
    const uint8_t *w[2 * V_TILES];
#pragma unroll
    for (int i = 0; i < 2 * V_TILES; i++) w[i] = p.w + (uint64_t)min(m0 + g + 8 * i, p.M - 1) * p.w_nb1 + t * 16;
    const uint8_t *x[NT];
    const float *xs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        x[n] = p.x + (uint64_t)min(n * 8 + g, p.N - 1) * p.x_nb1 + t * 16;
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
    for (int b0 = rank * V_WARPS + warp; b0 < whole; b0 += step * V_AHEAD) {
        uint4 a[V_AHEAD][2 * V_TILES][2], xv[V_AHEAD][NT][2];
        float s[V_AHEAD][NT][2];
#pragma unroll
        for (int i = 0; i < V_AHEAD; i++) {
            const int b = b0 + i * step;
            if (b >= whole) break;
#pragma unroll
            for (int r = 0; r < 2 * V_TILES; r++) {
                a[i][r][0] = ld_stream16(w[r] + (int64_t)b * F8B);
                a[i][r][1] = ld_stream16(w[r] + (int64_t)b * F8B + 64);
            }
        }
#pragma unroll
        for (int i = 0; i < V_AHEAD; i++) {
            const int b = b0 + i * step;
            if (b >= whole) break;
            const float sw = ws[b];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                xv[i][n][0] = *reinterpret_cast<const uint4 *>(x[n] + (int64_t)b * F8B);
                xv[i][n][1] = *reinterpret_cast<const uint4 *>(x[n] + (int64_t)b * F8B + 64);
                s[i][n][0] = xs[n][0][b] * sw;
                s[i][n][1] = xs[n][1][b] * sw;
            }
        }
#pragma unroll
        for (int i = 0; i < V_AHEAD; i++) {
            if (b0 + i * step >= whole) break;
            product(a[i], xv[i], s[i]);
        }
    }
    if (whole < kb && whole % step == rank * V_WARPS + warp) {  // the row's last, shorter block
        uint4 a[2 * V_TILES][2], xv[NT][2];
        float s[NT][2];
        const int k = whole * F8B, left = p.K - k - t * 16;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int n1 = left - 64 * h;
#pragma unroll
            for (int r = 0; r < 2 * V_TILES; r++) a[r][h] = ld_unit(w[r] + k + 64 * h, n1);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                xv[n][h] = ld_unit(x[n] + k + 64 * h, n1);
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

template <int NT, typename T>
int launch_v(const F8Gemm &p, int ctas, int splits, cudaStream_t s) {
    return launch_early("mul_mat_f8", gemv_f8_kernel<NT, T>, dim3((unsigned)ctas), dim3(32 * V_WARPS), 0, splits, s, p, splits);
}

}  // namespace

int gemv_f8_max_rows() { return 16; }

int launch_gemv_f8(const F8Gemm &p, cudaStream_t s) {
    const int64_t tiles = ((int64_t)p.M + V_ROWS - 1) / V_ROWS;
    const int kb = (p.K + F8B - 1) / F8B;
    // split the blocks until two CTAs per SM are busy, eight warps with a block each
    int splits = 1;
    while (splits < 8 && tiles * splits < 2 * sm_count() && kb >= 2 * splits * V_WARPS) splits *= 2;
    if (tiles * splits > INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, "mul_mat_f8: too many tiles");
    const int ctas = (int)(tiles * splits);
    const bool one = p.N <= 8;
    if (p.out_type == FB_F32) return one ? launch_v<1, float>(p, ctas, splits, s) : launch_v<2, float>(p, ctas, splits, s);
    if (p.out_type == FB_F16) return one ? launch_v<1, __half>(p, ctas, splits, s) : launch_v<2, __half>(p, ctas, splits, s);
    return one ? launch_v<1, __nv_bfloat16>(p, ctas, splits, s) : launch_v<2, __nv_bfloat16>(p, ctas, splits, s);
}

}  // namespace fbk
