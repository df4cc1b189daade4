// e4m3 matrix product for few rows of x (a decode step): the weights are read
// once, straight into tensor-core fragments.
//
// A warp takes 16 weight rows x one block of 128 values at a time: thread
// (g, t) of the m16n8k32 layout loads the 16-byte units t and t + 4 of rows g
// and g + 8. The layout's own order of k within a row does not matter to a
// sum as long as both operands use the same one, so two whole 16-byte loads
// serve four MMAs and nothing is shuffled. The products of a block are scaled
// in registers; the eight warps of a CTA take blocks in turn and meet in
// shared memory in warp order. Few weight rows: a cluster of S CTAs splits
// the blocks further and adds its partial sums in rank order through
// distributed shared memory.
//
// Bound by memory: one instruction in five is a load, each warp has four
// blocks (8 KB) in flight.
#include <cuda_runtime.h>

#include <algorithm>

#include "../host_common.h"
#include "gemm_f8.cuh"

namespace fbk {

namespace {

constexpr int V_WARPS = 8;
constexpr int V_ROWS = 16;   // weight rows per CTA
constexpr int V_AHEAD = 4;   // blocks in flight per warp

// The 16-byte unit at `p`, of which `n` bytes exist.
__device__ __forceinline__ uint4 ld_unit(const uint8_t *p, int n) {
    if (n >= 16) return ld_stream16(p);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < n; i++) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 ld_unit_cached(const uint8_t *p, int n) {
    if (n >= 16) return *reinterpret_cast<const uint4 *>(p);
    return ld_unit(p, n);
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
    const uint8_t *w0 = p.w + (uint64_t)min(m0 + g, p.M - 1) * p.w_nb1;
    const uint8_t *w1 = p.w + (uint64_t)min(m0 + g + 8, p.M - 1) * p.w_nb1;
    const uint8_t *x[NT];
    const float *xs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        x[n] = p.x + (uint64_t)min(n * 8 + g, p.N - 1) * p.x_nb1;
#pragma unroll
        for (int h = 0; h < 2; h++)
            xs[n][h] = reinterpret_cast<const float *>(p.xs + (uint64_t)min(n * 8 + 2 * t + h, p.N - 1) * p.xs_nb1);
    }
    const float *ws = reinterpret_cast<const float *>(p.ws + (uint64_t)(m0 / F8B) * p.ws_nb1);
    float acc[NT][4] = {};
    const int step = V_WARPS * splits;
    for (int b0 = rank * V_WARPS + warp; b0 < kb; b0 += step * V_AHEAD) {
        uint4 a[V_AHEAD][4];
        float s[V_AHEAD];
#pragma unroll
        for (int i = 0; i < V_AHEAD; i++) {
            const int b = b0 + i * step, k = b * F8B + t * 16;
            s[i] = 0.0f;
            if (b < kb) {
                const int n0 = p.K - k, n1 = p.K - k - 64;
                a[i][0] = ld_unit(w0 + k, n0);
                a[i][1] = ld_unit(w1 + k, n0);
                a[i][2] = ld_unit(w0 + k + 64, n1);
                a[i][3] = ld_unit(w1 + k + 64, n1);
                s[i] = ws[b];
            }
        }
#pragma unroll
        for (int i = 0; i < V_AHEAD; i++) {
            const int b = b0 + i * step, k = b * F8B + t * 16;
            if (b >= kb) break;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 x0 = ld_unit_cached(x[n] + k, p.K - k), x1 = ld_unit_cached(x[n] + k + 64, p.K - k - 64);
                float d[4] = {};
                mma_f8(d, {a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y}, x0.x, x0.y);
                mma_f8(d, {a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w}, x0.z, x0.w);
                mma_f8(d, {a[i][2].x, a[i][3].x, a[i][2].y, a[i][3].y}, x1.x, x1.y);
                mma_f8(d, {a[i][2].z, a[i][3].z, a[i][2].w, a[i][3].w}, x1.z, x1.w);
                const float s0 = xs[n][0][b] * s[i], s1 = xs[n][1][b] * s[i];
                acc[n][0] = fmaf(d[0], s0, acc[n][0]);
                acc[n][1] = fmaf(d[1], s1, acc[n][1]);
                acc[n][2] = fmaf(d[2], s0, acc[n][2]);
                acc[n][3] = fmaf(d[3], s1, acc[n][3]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int h = 0; h < 4; h++) part[warp][n * 8 + 2 * t + (h & 1)][g + (h >> 1) * 8] = acc[n][h];
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
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(32 * V_WARPS);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)splits;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemv_f8_kernel<NT, T>, p, splits);
    if (e != cudaSuccess) return fb::set_error(FB_ERR_CUDA, "mul_mat_f8 launch: %s", cudaGetErrorString(e));
    return FB_OK;
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
