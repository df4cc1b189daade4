// Shared by the e4m3 matrix products (gemm_f8.cu, gemv_f8.cu): operands,
// groups of rows, and the search of a work item's group.
//
//   out[n, m] = sum_b xs[n, b] * ws[m / 128, b] * (sum_{k in block b} x[n, k] * w[m, k])
//
// The inner sum is a tensor-core product accumulated in f32; its block scale
// and the sum over blocks are f32 operations outside the tensor core (two f32
// scales cannot be folded into e4m3 operands), in ascending b.
#pragma once

#include <cstdint>

#include "f8.cuh"
#include "kernels.h"

namespace fbk {

// One group's rows of a grouped product (the whole product when ungrouped).
struct F8Group {
    int expert, row0, rows;
};

// Group e, checked: a group that does not lie inside the n_rows rows of the
// output counts as empty (and is reported through status bit 1).
__device__ __forceinline__ F8Group f8_group(const F8Groups &g, int e, int32_t *status) {
    const int c = g.counts[e], o = g.offsets[e];
    if (c < 0 || o < 0 || c > g.n_rows || o > g.n_rows - c) {
        report_status(status, STATUS_BAD_ID);
        return {e, 0, 0};
    }
    return {e, o, c};
}

// Source row of grouped row r (r inside [0, n_rows)): -1 where the row table
// points outside the activations.
__device__ __forceinline__ int f8_source(const F8Groups &g, int r, int32_t *status) {
    if (!g.rows) return r;
    const int i = g.rows[r];
    const int t = i < 0 ? -1 : i / g.n_selected;
    if (t < 0 || t >= g.n_x) {
        report_status(status, STATUS_BAD_ID);
        return -1;
    }
    return t;
}

// The row of the caller's x behind grouped row r, as f8_source, whether the
// rows are gathered by the product itself or were beforehand.
__device__ __forceinline__ int f8_origin(const F8Groups &g, int r, int32_t *status) {
    if (!g.gathered) return f8_source(g, r, status);
    const int i = g.gathered[r];
    const int t = i < 0 ? -1 : i / g.n_selected;
    if (t < 0 || t >= g.n_origin) {
        report_status(status, STATUS_BAD_ID);
        return -1;
    }
    return t;
}

// The group and row tile (of `bm` rows) behind index `tile` when every group
// is cut into tiles of its own; expert < 0 past the last one. Called by a
// whole warp.
__device__ __forceinline__ F8Group f8_find_tile(const F8Groups &g, int tile, int bm, int32_t *status) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int e0 = 0; e0 < g.n_experts; e0 += 32) {
        F8Group f{-1, 0, 0};
        if (e0 + lane < g.n_experts) f = f8_group(g, e0 + lane, status);
        int run = (f.rows + bm - 1) / bm;
        const int mine = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        const bool hit = tile < before + run && tile >= before + run - mine;
        const unsigned who = __ballot_sync(0xffffffffu, hit);
        if (who) {
            const int src = __ffs(who) - 1;
            const int first = __shfl_sync(0xffffffffu, before + run - mine, src);
            const int at = (tile - first) * bm;
            const int r0 = __shfl_sync(0xffffffffu, f.row0, src), n = __shfl_sync(0xffffffffu, f.rows, src);
            return {e0 + src, r0 + at, min(bm, n - at)};
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
    return {-1, 0, 0};
}

// D += A * B^T for e4m3 fragments, m16n8k32, f32 accumulators.
__device__ __forceinline__ void mma_f8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace fbk
