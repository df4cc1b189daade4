// e4m3 matrix product for operands of any alignment and stride (rows that do
// not start on 16-byte boundaries cannot be fetched by TMA). 64 x 64 output
// tiles, four warps of 32 x 32; one block of 128 values per step, staged
// through shared memory with whatever alignment the rows have, multiplied
// with m16n8k32 tensor-core instructions and scaled in f32. Bound by those
// (about 100 cycles each) and by staging, which nothing overlaps: 4096 x 4096
// with one row 354 us, 512 rows 780 us, 2048 rows 2.1 ms, where aligned rows
// take 5.5, 20 and 42 us.
#include <cuda_runtime.h>

#include "../host_common.h"
#include "gemm_f8.cuh"

namespace fbk {

namespace {

constexpr int AB = 64;          // tile rows and columns
constexpr int A_PITCH = 144;    // bytes per staged row: fragments of 8 rows fall into different banks
constexpr int A_THREADS = 128;

// Four bytes at any address; only the aligned words that hold one of the
// first `n` bytes are read, the rest is zero.
__device__ __forceinline__ uint32_t ld4_any(const uint8_t *p, int n) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const uint32_t *w = reinterpret_cast<const uint32_t *>(a & ~uintptr_t(3));
    const int sh = (int)(a & 3);
    const uint32_t w0 = w[0], w1 = sh + n > 4 ? w[1] : 0u;
    const uint32_t v = __funnelshift_r(w0, w1, sh * 8);
    return n >= 4 ? v : v & ((1u << (8 * n)) - 1u);
}

template <typename T>
__global__ void __launch_bounds__(A_THREADS) gemm_f8_any_kernel(const F8Gemm p) {
    __shared__ __align__(16) uint8_t sx[AB * A_PITCH], sw[AB * A_PITCH];
    __shared__ int src[AB];
    __shared__ F8Group s_grp;
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int64_t my = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;  // tile of weight rows
    if (my * AB >= p.M) return;
    const int m0 = (int)my * AB;
    F8Group grp{0, (int)blockIdx.x * AB, 0};
    if (p.g.counts) {
        if (warp == 0) {
            grp = f8_find_tile(p.g, blockIdx.x, AB, p.status);
            if (lane == 0) s_grp = grp;
        }
        __syncthreads();
        grp = s_grp;
        if (grp.expert < 0) return;
        if (blockIdx.x == gridDim.x - 1) {  // a tile that groups which do not overlap never have
            if (tid == 0) report_status(p.status, STATUS_BAD_ID);
            return;
        }
    } else {
        grp.rows = min(AB, p.N - grp.row0);
    }
    if (tid < AB) src[tid] = tid < grp.rows ? (p.g.counts ? f8_source(p.g, grp.row0 + tid, p.status) : grp.row0 + tid) : -1;
    __syncthreads();
    const uint8_t *w = p.w + (uint64_t)grp.expert * p.w_nb2;
    const uint8_t *ws = p.ws + (uint64_t)grp.expert * p.ws_nb2;
    const int wm = (warp & 1) * 32, wn = (warp >> 1) * 32;  // this warp's tokens, weight rows
    const float *xsr[4];  // scale rows of the four token rows a thread accumulates
    bool live[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = src[wm + (i >> 1) * 16 + (i & 1) * 8 + g];
        live[i] = r >= 0;
        xsr[i] = reinterpret_cast<const float *>(p.xs + (uint64_t)max(r, 0) * p.xs_nb1);
    }
    float acc[2][4][4] = {};
    const int kb = (p.K + F8B - 1) / F8B;
    for (int b = 0; b < kb; b++) {
        for (int i = tid; i < 2 * AB * (F8B / 4); i += A_THREADS) {
            const int c = i % (F8B / 4), r = i / (F8B / 4) % AB, k = b * F8B + c * 4;
            const bool is_w = i >= AB * (F8B / 4);
            const int row = is_w ? m0 + r : src[r];
            const bool in = k < p.K && (is_w ? row < p.M : row >= 0);
            const uint8_t *a = is_w ? w + (uint64_t)row * p.w_nb1 + k : p.x + (uint64_t)row * p.x_nb1 + k;
            *reinterpret_cast<uint32_t *>((is_w ? sw : sx) + r * A_PITCH + c * 4) = in ? ld4_any(a, min(4, p.K - k)) : 0u;
        }
        __syncthreads();
        float part[2][4][4] = {};
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            uint32_t a[2][4];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int h = 0; h < 4; h++)
                    a[i][h] = *reinterpret_cast<const uint32_t *>(sx + (wm + i * 16 + (h & 1) * 8 + g) * A_PITCH + kk * 32 +
                                                                  (h >> 1) * 16 + t * 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t *bp = sw + (wn + j * 8 + g) * A_PITCH + kk * 32 + t * 4;
                const uint32_t b0 = *reinterpret_cast<const uint32_t *>(bp), b1 = *reinterpret_cast<const uint32_t *>(bp + 16);
#pragma unroll
                for (int i = 0; i < 2; i++) mma_f8(part[i][j], a[i], b0, b1);
            }
        }
        // the tile's weight rows lie in one block row: 64 divides 128
        const float wsc = reinterpret_cast<const float *>(ws + (uint64_t)(m0 / F8B) * p.ws_nb1)[b];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float sc = live[i] ? xsr[i][b] * wsc : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                acc[i >> 1][j][(i & 1) * 2] = fmaf(part[i >> 1][j][(i & 1) * 2], sc, acc[i >> 1][j][(i & 1) * 2]);
                acc[i >> 1][j][(i & 1) * 2 + 1] = fmaf(part[i >> 1][j][(i & 1) * 2 + 1], sc, acc[i >> 1][j][(i & 1) * 2 + 1]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = wm + (i >> 1) * 16 + (i & 1) * 8 + g;
        if (r >= grp.rows) continue;
        T *o = reinterpret_cast<T *>(p.y + (uint64_t)(grp.row0 + r) * p.y_nb1);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int m = m0 + wn + j * 8 + t * 2 + h;
                if (m < p.M) o[m] = from_f32<T>(live[i] ? acc[i >> 1][j][(i & 1) * 2 + h] : 0.0f);
            }
    }
}

}  // namespace

int launch_gemm_f8_any(const F8Gemm &p, cudaStream_t s) {
    // every group's last tile may be a partial one, which makes fewer tiles than
    // this: the last index is left for groups that overlap
    const int64_t gx = ((int64_t)p.N + AB - 1) / AB + (p.g.counts ? p.g.n_experts : 0);
    const int64_t tiles = ((int64_t)p.M + AB - 1) / AB, gz = (tiles + 65534) / 65535;  // grid.y has 16 bits
    const dim3 grid((unsigned)gx, (unsigned)((tiles + gz - 1) / gz), (unsigned)gz);
    const char *what = "mul_mat_f8";
    if (p.out_type == FB_F32) return launch_early(what, gemm_f8_any_kernel<float>, grid, dim3(A_THREADS), 0, 1, s, p);
    if (p.out_type == FB_F16) return launch_early(what, gemm_f8_any_kernel<__half>, grid, dim3(A_THREADS), 0, 1, s, p);
    return launch_early(what, gemm_f8_any_kernel<__nv_bfloat16>, grid, dim3(A_THREADS), 0, 1, s, p);
}

}  // namespace fbk
