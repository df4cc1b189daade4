// Row operators that end in the e4m3 form (f8.cuh): plain quantization of
// activations, silu(gate) * up, rms_norm with the residual's addition, and
// the quantization of a weight matrix in 128 x 128 blocks.
//
// All of them are bound by memory: a few operations per byte, every value
// read once and written once. The block maximum is taken of values that stay
// in registers between the load and the store, so no operator makes a second
// pass over its input (but the norm of rows that are aligned to less than 16
// bytes or too long for registers: norm_f8_any_kernel).
#include <cuda_runtime.h>

#include <algorithm>

#include "../host_common.h"
#include "f8.cuh"
#include "kernels.h"

namespace fbk {

namespace {

// ---------------------------------------------------------------------------
// quantize (one operand) and silu_mul (two): blocks are independent. A block
// of 128 values belongs to G consecutive lanes that hold one 32-byte vector
// each (G = 8 for 16-bit types, 16 for f32); its maximum is a shuffle
// reduction over them. 16-byte vectors where rows or pointers are aligned to
// no more (half the bytes in flight: bf16 8192 x 4096 took 25.1 us, not
// 17.9); a warp per block with single-element accesses where to less, lane l
// elements l, l + 32, ...
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

struct RowParams {
    const uint8_t *x, *y;  // y: up (silu_mul)
    uint64_t x_nb1, y_nb1;
    uint8_t *q;
    uint64_t q_nb1;
    uint8_t *s;
    uint64_t s_nb1;
    int64_t total;  // rows * blocks per row
    int64_t k;
    uint32_t kb;    // blocks per row
    uint32_t kb_mul, kb_shift;  // n / kb = (mulhi(n, kb_mul) + n) >> kb_shift, n < 2^31
};

// silu(g) * u = g (u / (1 + e^-g)). The exponential and the reciprocal are the
// fast forms: with the exact ones the kernel is bound by arithmetic instead of
// memory. The exponential is off by 3 + |g| units in the last place of f32, the
// result goes to 4 significant bits. u is multiplied first: by at most 1, and a
// subnormal gate keeps its bits. For gates down to kSiluNear, where e^-g and
// its reciprocal are normal numbers.
constexpr float kSiluNear = -87.0f;
__device__ __forceinline__ float silu_mul_near(float g, float u) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * (r * u);
}
// Any gate: (g t) (t u) / (16 + t^2) with t = 4 e^(g/2) for g < 0. As one factor
// e^g leaves the normal range below -87, where a large u brings the product
// back; in two halves it does not before the product is below what a block
// rounds to zero (g = -177).
__device__ __forceinline__ float silu_mul_any(float g, float u) {
    if (!(g < 0.0f)) return silu_mul_near(g, u);
    float t, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(g, 0.72134752f, 2.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(t, t, 16.0f)));
    return (g * t) * (t * r * u);
}

// Whether a vector holds a gate below kSiluNear (or a negative NaN): their bits
// are above those of kSiluNear as unsigned numbers, all others below or equal.
// A quarter of an instruction per 16-bit value.
template <typename T, int H>
__device__ __forceinline__ bool silu_far(const uint4 (&v)[H]) {
    uint32_t m = 0;
#pragma unroll
    for (int h = 0; h < H; h++) {
        if constexpr (sizeof(T) == 4)
            m = __vimax3_u32(__vimax3_u32(m, v[h].x, v[h].y), v[h].z, v[h].w);
        else
            m = __vimax3_u16x2(__vimax3_u16x2(m, v[h].x, v[h].y), v[h].z, v[h].w);
    }
    if constexpr (sizeof(T) == 4) return m > __float_as_uint(kSiluNear);
    constexpr uint32_t near = std::is_same<T, __half>::value ? 0xd570u : 0xc2aeu;  // -87 in f16, bf16
    return (m >> 16) > near || (m & 0xffffu) > near;
}

// W: bytes per lane and operand, 32 or 16, or 0 for single elements.
template <typename T, bool SILU, int W>
__global__ void __launch_bounds__(kRowThreads, 2048 / kRowThreads) rows_f8_kernel(const RowParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    constexpr int N = W ? W / (int)sizeof(T) : 4;
    constexpr int G = F8B / N;
    constexpr int V = Vec<T>::N;
    const int lane = threadIdx.x % G;
    const int64_t gid = (int64_t)blockIdx.x * (kRowThreads / G) + threadIdx.x / G;
    const bool live = gid < p.total;
    // the division by the blocks per row: by a multiplication where the count
    // fits 31 bits
    int64_t row;
    uint32_t b;
    if (p.total <= 0x7fffffff) {
        row = (__umulhi((uint32_t)gid, p.kb_mul) + (uint32_t)gid) >> p.kb_shift;
        b = (uint32_t)gid - (uint32_t)row * p.kb;
    } else {
        row = gid / p.kb;
        b = (uint32_t)(gid - row * p.kb);
    }
    const int64_t k0 = (int64_t)b * F8B;
    const uint8_t *xr = p.x + row * p.x_nb1;
    const uint8_t *yr = SILU ? p.y + row * p.y_nb1 : nullptr;
    float f[N];
    uint32_t top = 0;
    // (A lane that holds a far gate takes the form for any gate. That branch
    // stands ahead of all arithmetic, and the launch bound holds the kernel to 32
    // registers, full occupancy: bf16 4096 x 11008 35.4 us. With 40 registers
    // 37.3, with the branch behind the near products 35.9, with the form for any
    // gate throughout 40.4, without far gates 35.2.)
    if constexpr (W != 0) {
        const int64_t k = k0 + lane * N;  // k % N == 0 here: a vector lies inside the row or outside
        if (live && k < p.k) {
            uint4 v[N / V], u[N / V];
            if constexpr (W == 32) {
                const Wide32 a = ld_stream32(xr + k * sizeof(T));
                v[0] = a.lo;
                v[N / V - 1] = a.hi;
                if constexpr (SILU) {
                    const Wide32 c = ld_stream32(yr + k * sizeof(T));
                    u[0] = c.lo;
                    u[N / V - 1] = c.hi;
                }
            } else {
                v[0] = ld_stream16(xr + k * sizeof(T));
                if constexpr (SILU) u[0] = ld_stream16(yr + k * sizeof(T));
            }
            bool far = false;
            if constexpr (SILU) far = silu_far<T>(v);
            if (SILU && far) {
#pragma unroll
                for (int h = 0; h < N / V; h++) {
                    float x[V], y[V];
                    Vec<T>::get(v[h], x);
                    Vec<T>::get(u[h], y);
#pragma unroll
                    for (int i = 0; i < V; i++) f[h * V + i] = silu_mul_any(x[i], y[i]);
                }
            } else {
#pragma unroll
                for (int h = 0; h < N / V; h++) {
                    float x[V];
                    Vec<T>::get(v[h], x);
                    if constexpr (SILU) {
                        float y[V];
                        Vec<T>::get(u[h], y);
#pragma unroll
                        for (int i = 0; i < V; i++) x[i] = silu_mul_near(x[i], y[i]);
                    }
#pragma unroll
                    for (int i = 0; i < V; i++) f[h * V + i] = x[i];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) f[i] = 0.0f;
        }
    } else {
        float least = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int64_t k = k0 + lane + i * 32;
            f[i] = 0.0f;
            if (live && k < p.k) {
                f[i] = to_f32(reinterpret_cast<const T *>(xr)[k]);
                if constexpr (SILU) {
                    least = fminf(least, f[i]);
                    f[i] = silu_mul_near(f[i], to_f32(reinterpret_cast<const T *>(yr)[k]));
                }
            }
        }
        if (SILU && least < kSiluNear) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int64_t k = k0 + lane + i * 32;
                if (k < p.k) f[i] = silu_mul_any(to_f32(reinterpret_cast<const T *>(xr)[k]), to_f32(reinterpret_cast<const T *>(yr)[k]));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) top = max(top, abs_bits(f[i]));
#pragma unroll
    for (int o = 1; o < G; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    float s, r;
    f8_scale(top, s, r);
    if (!live) return;
    uint8_t *qr = p.q + row * p.q_nb1;
    if constexpr (W != 0) {
        const int64_t k = k0 + lane * N;
        if (k < p.k) {
            uint32_t w[N / 4];
#pragma unroll
            for (int i = 0; i < N / 4; i++) w[i] = f8_pack4(f[4 * i] * r, f[4 * i + 1] * r, f[4 * i + 2] * r, f[4 * i + 3] * r);
            if constexpr (N == 16)
                *reinterpret_cast<uint4 *>(qr + k) = make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (N == 8)
                *reinterpret_cast<uint2 *>(qr + k) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t *>(qr + k) = w[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int64_t k = k0 + lane + i * 32;
            if (k < p.k) qr[k] = f8_one(f[i] * r);
        }
    }
    if (lane == 0) reinterpret_cast<float *>(p.s + row * p.s_nb1)[b] = s;
}

// ---------------------------------------------------------------------------
// Weights: one CTA per 128 x 128 block, its values in registers.
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 512;

struct TileParams {
    const uint8_t *x;
    uint64_t x_nb1;
    uint8_t *q;
    uint64_t q_nb1;
    uint8_t *s;
    uint64_t s_nb1;
    int64_t rows, k;
    uint32_t kb;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kTileThreads) tile_f8_kernel(const TileParams p) {
    constexpr int N = VEC ? Vec<T>::N : 1;
    constexpr int G = F8B / N;                  // threads per row
    constexpr int RS = kTileThreads / G;        // rows per step
    constexpr int STEPS = F8B / RS;
    __shared__ uint32_t s_top[kTileThreads / 32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t br = blockIdx.x / p.kb;
    const uint32_t bc = (uint32_t)(blockIdx.x - br * p.kb);
    const int64_t k = (int64_t)bc * F8B + (threadIdx.x % G) * N;
    const int64_t row0 = br * F8B + threadIdx.x / G;
    const bool in_k = k < p.k;
    uint4 v[VEC ? STEPS : 1];
    float e[VEC ? 1 : STEPS];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int64_t row = row0 + i * RS;
        const bool in = in_k && row < p.rows;
        const uint8_t *a = p.x + row * p.x_nb1 + k * sizeof(T);
        if constexpr (VEC)
            v[i] = in ? ld_stream16(a) : make_uint4(0, 0, 0, 0);
        else
            e[i] = in ? to_f32(*reinterpret_cast<const T *>(a)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        if constexpr (VEC) {
            float f[N];
            Vec<T>::get(v[i], f);
#pragma unroll
            for (int j = 0; j < N; j++) top = max(top, abs_bits(f[j]));
        } else {
            top = max(top, abs_bits(e[i]));
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, s_top[threadIdx.x % (kTileThreads / 32)]);
    float s, r;
    f8_scale(top, s, r);
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int64_t row = row0 + i * RS;
        if (!in_k || row >= p.rows) continue;
        uint8_t *q = p.q + row * p.q_nb1 + k;
        if constexpr (VEC) {
            float f[N];
            Vec<T>::get(v[i], f);
            const uint32_t lo = f8_pack4(f[0] * r, f[1] * r, f[2] * r, f[3] * r);
            if constexpr (N == 8) {
                const uint32_t hi = f8_pack4(f[4] * r, f[5] * r, f[6] * r, f[7] * r);
                *reinterpret_cast<uint2 *>(q) = make_uint2(lo, hi);
            } else {
                *reinterpret_cast<uint32_t *>(q) = lo;
            }
        } else {
            *q = f8_one(e[i] * r);
        }
    }
    if (threadIdx.x == 0) reinterpret_cast<float *>(p.s + br * p.s_nb1)[bc] = s;
}

// ---------------------------------------------------------------------------
// rms_norm: h = round(x + residual) is stored and kept in registers as it is
// stored (so the fused call gives the bits of an addition followed by the
// norm), y = (h * (1 / sqrt(mean(h^2) + eps))) * weight goes to the 8-bit
// form. The sum of squares is held in f32 in a fixed order.
// ---------------------------------------------------------------------------
struct NormF8Params {
    const uint8_t *x, *res, *w;
    uint64_t x_nb1, res_nb1;
    uint8_t *sum;
    uint64_t sum_nb1;
    uint8_t *q;
    uint64_t q_nb1;
    uint8_t *s;
    uint64_t s_nb1;
    int64_t rows, k;
    float eps;
    int w_f32;  // weight in f32 (else in the type of x)
};

// Sum over the CTA's warps, in warp order; the same value in every thread.
__device__ __forceinline__ float cta_sum(float v, float *part) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
    return warp_sum(lane < nw ? part[lane] : 0.0f);
}

// W bytes (16 or 32) of a row as 16-byte vectors, and back.
template <int W>
__device__ __forceinline__ void ld_wide(uint4 (&v)[W / 16], const void *p) {
    if constexpr (W == 32) {
        const Wide32 a = ld_stream32(p);
        v[0] = a.lo;
        v[1] = a.hi;
    } else {
        v[0] = ld_stream16(p);
    }
}
template <int W>
__device__ __forceinline__ void st_wide(void *p, const uint4 (&v)[W / 16]) {
#pragma unroll
    for (int i = 0; i < W / 16; i++) reinterpret_cast<uint4 *>(p)[i] = v[i];
}

// The row in registers: NV vectors of W bytes per thread. WARP: a warp per
// row (blockDim.y rows per CTA), else a CTA per row. (The bound of 1024 threads
// holds NV = 4 at W = 32 to 64 registers; the 16-bit types spill 152 bytes
// there. It takes rows of more than 32 KB, or 64 KB where rows are few.)
template <typename T, int NV, bool WARP, int W>
__global__ void __launch_bounds__(WARP ? 256 : 1024) norm_f8_kernel(const NormF8Params p) {
    constexpr int V = Vec<T>::N, H = W / 16, N = V * H, G = F8B / N;
    __shared__ float part[32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t row = WARP ? (int64_t)blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x;
    if (WARP && row >= p.rows) return;
    const int t = threadIdx.x, nt = WARP ? 32 : blockDim.x;
    const uint8_t *xr = p.x + row * p.x_nb1;
    uint4 v[NV][H];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t k = (int64_t)(i * nt + t) * N;
#pragma unroll
        for (int h = 0; h < H; h++) v[i][h] = make_uint4(0, 0, 0, 0);
        if (k < p.k) ld_wide<W>(v[i], xr + k * sizeof(T));
    }
    if (p.res) {
        const uint8_t *rr = p.res + row * p.res_nb1;
        uint8_t *hr = p.sum + row * p.sum_nb1;
        uint4 u[NV][H];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int64_t k = (int64_t)(i * nt + t) * N;
#pragma unroll
            for (int h = 0; h < H; h++) u[i][h] = make_uint4(0, 0, 0, 0);
            if (k < p.k) ld_wide<W>(u[i], rr + k * sizeof(T));
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int64_t k = (int64_t)(i * nt + t) * N;
#pragma unroll
            for (int h = 0; h < H; h++) {
                float a[V], b[V];
                Vec<T>::get(v[i][h], a);
                Vec<T>::get(u[i][h], b);
#pragma unroll
                for (int j = 0; j < V; j++) a[j] += b[j];
                v[i][h] = Vec<T>::put(a);
            }
            if (k < p.k) st_wide<W>(hr + k * sizeof(T), v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int h = 0; h < H; h++) {
            float f[V];
            Vec<T>::get(v[i][h], f);
#pragma unroll
            for (int j = 0; j < V; j++) ss = fmaf(f[j], f[j], ss);
        }
    ss = WARP ? warp_sum(ss) : cta_sum(ss, part);
    const float inv = 1.0f / sqrtf(ss / (float)p.k + p.eps);
    uint8_t *qr = p.q + row * p.q_nb1;
    float *sr = reinterpret_cast<float *>(p.s + row * p.s_nb1);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int64_t k = (int64_t)(i * nt + t) * N;
        const bool in = k < p.k;
        float f[N];
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < H; h++) {
            float x[V];
            Vec<T>::get(v[i][h], x);
            if (in) {
                float g[V];
                if (sizeof(T) == 4 || !p.w_f32) {
                    Vec<T>::get(__ldg(reinterpret_cast<const uint4 *>(p.w + (k + h * V) * sizeof(T))), g);
                } else {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float4 w4 = __ldg(reinterpret_cast<const float4 *>(p.w + (k + h * V + j) * 4));
                        g[j] = w4.x;
                        g[j + 1] = w4.y;
                        g[j + 2] = w4.z;
                        g[j + 3] = w4.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    x[j] = x[j] * inv * g[j];
                    top = max(top, abs_bits(x[j]));
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) f[h * V + j] = x[j];
        }
#pragma unroll
        for (int o = 1; o < G; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        float s, r;
        f8_scale(top, s, r);
        if (in) {
            uint32_t w[N / 4];
#pragma unroll
            for (int j = 0; j < N / 4; j++) w[j] = f8_pack4(f[4 * j] * r, f[4 * j + 1] * r, f[4 * j + 2] * r, f[4 * j + 3] * r);
            if constexpr (N == 16)
                *reinterpret_cast<uint4 *>(qr + k) = make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (N == 8)
                *reinterpret_cast<uint2 *>(qr + k) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t *>(qr + k) = w[0];
            if (t % G == 0) sr[k / F8B] = s;
        }
    }
}

// Rows of any length and alignment: the sum of squares in one pass, the norm
// in a second one that reads the stored sum (or x) again, a warp per block.
// (A variant that held such rows in registers took 1.6 times as long at 4001 x
// 4101 bf16: single elements need the occupancy more than the saved pass.) With
// a residual that takes 79 us, four times what the bytes take at the copy rate.
template <typename T>
__global__ void __launch_bounds__(1024) norm_f8_any_kernel(const NormF8Params p) {
    __shared__ float part[32];
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t row = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(p.x + row * p.x_nb1);
    const T *res = p.res ? reinterpret_cast<const T *>(p.res + row * p.res_nb1) : nullptr;
    T *sum = p.res ? reinterpret_cast<T *>(p.sum + row * p.sum_nb1) : nullptr;
    float ss = 0.0f;
    for (int64_t k = threadIdx.x; k < p.k; k += blockDim.x) {
        float f = to_f32(x[k]);
        if (res) {
            const T h = from_f32<T>(f + to_f32(res[k]));
            sum[k] = h;
            f = to_f32(h);
        }
        ss = fmaf(f, f, ss);
    }
    ss = cta_sum(ss, part);  // its barrier also orders the stored sums before the reads below
    const float inv = 1.0f / sqrtf(ss / (float)p.k + p.eps);
    const T *h = res ? sum : x;
    const int lane = threadIdx.x & 31;
    uint8_t *qr = p.q + row * p.q_nb1;
    float *sr = reinterpret_cast<float *>(p.s + row * p.s_nb1);
    for (int64_t b = threadIdx.x >> 5; b * F8B < p.k; b += blockDim.x >> 5) {
        float f[4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t k = b * F8B + lane + i * 32;
            f[i] = 0.0f;
            if (k < p.k) {
                const float g = p.w_f32 ? reinterpret_cast<const float *>(p.w)[k] : to_f32(reinterpret_cast<const T *>(p.w)[k]);
                f[i] = to_f32(h[k]) * inv * g;
            }
            top = max(top, abs_bits(f[i]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        float s, r;
        f8_scale(top, s, r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t k = b * F8B + lane + i * 32;
            if (k < p.k) qr[k] = f8_one(f[i] * r);
        }
        if (lane == 0) sr[b] = s;
    }
}

bool aligned(uint64_t a, const void *p, uint64_t nb1) { return ((reinterpret_cast<uintptr_t>(p) | nb1) & (a - 1)) == 0; }

template <typename T, bool SILU>
int launch_rows_t(const RowParams &p, int width, cudaStream_t s, const char *what) {
    const int groups = kRowThreads / (width ? F8B / (width / (int)sizeof(T)) : 32);
    const int64_t grid = (p.total + groups - 1) / groups;
    if (grid > INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, "%s: too many blocks", what);
    auto *fn = width == 32 ? rows_f8_kernel<T, SILU, 32> : width == 16 ? rows_f8_kernel<T, SILU, 16> : rows_f8_kernel<T, SILU, 0>;
    return launch_early(what, fn, dim3((unsigned)grid), dim3(kRowThreads), 0, 1, s, p);
}

template <typename T, int W>
int launch_norm_w(const NormF8Params &p, cudaStream_t s) {
    const char *what = "rms_norm_f8";
    const int64_t vecs = p.k / (W / (int)sizeof(T));
    // A warp per row for short rows in numbers that fill the GPU; else a CTA
    // per row: one vector per thread when rows are few (latency), more
    // vectors and smaller CTAs when they are many (2048 rows of 16384 f16:
    // 41.4 us with 512 threads, 47.6 with 256, 49.7 with 1024).
    if (vecs <= 64 && p.rows >= 1024) {
        auto *fn = vecs <= 32 ? norm_f8_kernel<T, 1, true, W> : norm_f8_kernel<T, 2, true, W>;
        return launch_early(what, fn, dim3((unsigned)((p.rows + 7) / 8)), dim3(32, 8), 0, 1, s, p);
    }
    const int most = p.rows <= 2 * sm_count() ? 1024 : 512;
    int nv = 1;
    while (nv < 4 && (vecs + nv - 1) / nv > most) nv *= 2;
    const int threads = (int)(((vecs + nv - 1) / nv + 31) / 32 * 32);
    auto *fn = nv == 1 ? norm_f8_kernel<T, 1, false, W> : nv == 2 ? norm_f8_kernel<T, 2, false, W> : norm_f8_kernel<T, 4, false, W>;
    return launch_early(what, fn, dim3((unsigned)p.rows), dim3(threads), 0, 1, s, p);
}

// `width`: bytes that rows and pointers are aligned to, 32, 16 or 0.
template <typename T>
int launch_norm_t(const NormF8Params &p, int width, cudaStream_t s) {
    if (width == 32 && p.k * (int64_t)sizeof(T) <= 32 * 4 * 1024) return launch_norm_w<T, 32>(p, s);
    if (width && p.k * (int64_t)sizeof(T) <= 16 * 4 * 1024) return launch_norm_w<T, 16>(p, s);
    const int threads = (int)std::min<int64_t>(1024, (p.k + 31) / 32 * 32);
    return launch_early("rms_norm_f8", norm_f8_any_kernel<T>, dim3((unsigned)p.rows), dim3(threads), 0, 1, s, p);
}

int esize(int32_t type) { return type == FB_F32 ? 4 : 2; }

}  // namespace

int launch_rows_f8(int32_t type, const void *x, uint64_t x_nb1, const void *up, uint64_t up_nb1, int64_t rows,
                   int64_t k, const F8Out &o, cudaStream_t s) {
    const char *what = up ? "silu_mul_f8" : "quantize_f8";
    RowParams p{};
    p.x = static_cast<const uint8_t *>(x);
    p.x_nb1 = x_nb1;
    p.y = static_cast<const uint8_t *>(up);
    p.y_nb1 = up_nb1;
    p.q = static_cast<uint8_t *>(o.q);
    p.q_nb1 = o.q_nb1;
    p.s = reinterpret_cast<uint8_t *>(o.scale);
    p.s_nb1 = o.scale_nb1;
    p.k = k;
    p.kb = (uint32_t)((k + F8B - 1) / F8B);
    p.total = rows * p.kb;
    while ((1ull << p.kb_shift) < p.kb) p.kb_shift++;
    p.kb_mul = (uint32_t)(((1ull << 32) * ((1ull << p.kb_shift) - p.kb)) / p.kb + 1);
    auto fits = [&](int w) {
        const int n = w / esize(type);
        return k % n == 0 && aligned(w, x, x_nb1) && (!up || aligned(w, up, up_nb1)) && aligned(n, o.q, o.q_nb1);
    };
    const int vec = fits(32) ? 32 : fits(16) ? 16 : 0;
    switch (type) {
        case FB_F32:
            return up ? launch_rows_t<float, true>(p, vec, s, what) : launch_rows_t<float, false>(p, vec, s, what);
        case FB_F16:
            return up ? launch_rows_t<__half, true>(p, vec, s, what) : launch_rows_t<__half, false>(p, vec, s, what);
        default:
            return up ? launch_rows_t<__nv_bfloat16, true>(p, vec, s, what)
                      : launch_rows_t<__nv_bfloat16, false>(p, vec, s, what);
    }
}

int launch_quantize_f8_tiles(int32_t type, const void *x, uint64_t x_nb1, int64_t rows, int64_t k, const F8Out &o,
                             cudaStream_t s) {
    TileParams p{};
    p.x = static_cast<const uint8_t *>(x);
    p.x_nb1 = x_nb1;
    p.q = static_cast<uint8_t *>(o.q);
    p.q_nb1 = o.q_nb1;
    p.s = reinterpret_cast<uint8_t *>(o.scale);
    p.s_nb1 = o.scale_nb1;
    p.rows = rows;
    p.k = k;
    p.kb = (uint32_t)((k + F8B - 1) / F8B);
    const int64_t grid = (rows + F8B - 1) / F8B * p.kb;
    if (grid > INT32_MAX) return fb::set_error(FB_ERR_UNSUPPORTED, "quantize_f8: too many blocks");
    const int n = 16 / esize(type);
    const bool vec = k % n == 0 && aligned(16, x, x_nb1) && aligned(n, o.q, o.q_nb1);
    auto *fn = type == FB_F32   ? (vec ? tile_f8_kernel<float, true> : tile_f8_kernel<float, false>)
               : type == FB_F16 ? (vec ? tile_f8_kernel<__half, true> : tile_f8_kernel<__half, false>)
                                : (vec ? tile_f8_kernel<__nv_bfloat16, true> : tile_f8_kernel<__nv_bfloat16, false>);
    return launch_early("quantize_f8", fn, dim3((unsigned)grid), dim3(kTileThreads), 0, 1, s, p);
}

int launch_rms_norm_f8(int32_t type, const void *x, uint64_t x_nb1, const void *residual, uint64_t residual_nb1,
                       void *sum, uint64_t sum_nb1, int32_t wtype, const void *weight, float eps, int64_t rows,
                       int64_t k, const F8Out &o, cudaStream_t s) {
    NormF8Params p{};
    p.x = static_cast<const uint8_t *>(x);
    p.x_nb1 = x_nb1;
    p.res = static_cast<const uint8_t *>(residual);
    p.res_nb1 = residual_nb1;
    p.sum = static_cast<uint8_t *>(sum);
    p.sum_nb1 = sum_nb1;
    p.w = static_cast<const uint8_t *>(weight);
    p.w_f32 = wtype == FB_F32;
    p.q = static_cast<uint8_t *>(o.q);
    p.q_nb1 = o.q_nb1;
    p.s = reinterpret_cast<uint8_t *>(o.scale);
    p.s_nb1 = o.scale_nb1;
    p.rows = rows;
    p.k = k;
    p.eps = eps;
    auto fits = [&](int w) {
        const int n = w / esize(type);
        return k % n == 0 && aligned(w, x, x_nb1) && aligned(16, weight, 0) &&
               (!residual || (aligned(w, residual, residual_nb1) && aligned(16, sum, sum_nb1))) && aligned(n, o.q, o.q_nb1);
    };
    const int vec = fits(32) ? 32 : fits(16) ? 16 : 0;
    switch (type) {
        case FB_F32: return launch_norm_t<float>(p, vec, s);
        case FB_F16: return launch_norm_t<__half>(p, vec, s);
        default: return launch_norm_t<__nv_bfloat16>(p, vec, s);
    }
}

}  // namespace fbk
