// C entry points of the e4m3 operators: argument checks and the choice of
// kernel. Nothing is read or written on the device before every check has
// passed.
#include <cuda_runtime.h>

#include <cstdint>

#include "host_common.h"
#include "kernels/kernels.h"

using fb::set_error;

namespace {

constexpr int64_t kB = 128;  // values per scale
constexpr int64_t kMaxF8Experts = 1024;

int64_t esize(int32_t type) { return type == FB_F32 ? 4 : type == FB_F16 || type == FB_BF16 ? 2 : 0; }

bool off(const void *p, uint64_t nb, uint64_t a) { return ((reinterpret_cast<uintptr_t>(p) | nb) & (a - 1)) != 0; }

// A matrix of `rows` contiguous rows of `bytes` bytes: present, aligned to
// its elements, rows apart from one another.
int check_rows(const char *op, const char *name, const void *p, uint64_t nb1, int64_t rows, int64_t bytes, int64_t align) {
    if (!p) return set_error(FB_ERR_INVALID, "%s: %s is null", op, name);
    if (off(p, rows > 1 ? nb1 : 0, (uint64_t)align))
        return set_error(FB_ERR_INVALID, "%s: %s is not aligned to its elements", op, name);
    if (rows > 1 && nb1 < (uint64_t)bytes)
        return set_error(FB_ERR_SHAPE, "%s: rows of %s overlap (stride %llu, %lld bytes)", op, name,
                         (unsigned long long)nb1, (long long)bytes);
    return FB_OK;
}

#define FB_TRY(call)            \
    do {                        \
        const int rc_ = (call); \
        if (rc_) return rc_;    \
    } while (0)

int check_type(const char *op, int32_t type) {
    if (!esize(type)) return set_error(FB_ERR_UNSUPPORTED, "%s: type %d (F32, F16 and BF16)", op, type);
    return FB_OK;
}

int check_dims(const char *op, int64_t a, int64_t b, int64_t c) {
    if (a < 0 || b < 0 || c < 0) return set_error(FB_ERR_INVALID, "%s: negative dimension", op);
    constexpr int64_t most = INT32_MAX - 1024;  // a tile's end still fits an int
    if (a > most || b > most || c > most) return set_error(FB_ERR_UNSUPPORTED, "%s: dimension over 2^31 - 1025", op);
    return FB_OK;
}

// 8-bit output rows and their scales.
int check_out(const char *op, const fbk::F8Out &o, int64_t rows, int64_t k, int64_t scale_rows) {
    FB_TRY(check_rows(op, "q", o.q, o.q_nb1, rows, k, 1));
    return check_rows(op, "scale", o.scale, o.scale_nb1, scale_rows, (k + kB - 1) / kB * 4, 4);
}

// A row stride that no second row uses must not decide alignment.
uint64_t stride_of(uint64_t nb1, int64_t rows, int64_t bytes) { return rows > 1 ? nb1 : (uint64_t)(bytes + 15) / 16 * 16; }

int run_product(fbk::F8Gemm &p, void *ws, uint64_t ws_bytes, cudaStream_t s) {
    if (!fbk::gemm_f8_supported(p)) return fbk::launch_gemm_f8_any(p, s);
    if (!p.g.counts && p.N <= fbk::gemv_f8_max_rows()) return fbk::launch_gemv_f8(p, s);
    if (p.g.rows && fbk::gather_f8_pays(p.g.n_rows, p.g.n_experts) && ws && !off(ws, 0, 16) &&
        ws_bytes >= fbk::gather_f8_bytes(p.K, p.g.n_rows))
        FB_TRY(fbk::launch_gather_f8(p, ws, s));
    return fbk::launch_gemm_f8(p, s);
}

// K = 0: every sum is empty.
int zero_rows(const char *op, void *dst, uint64_t dst_nb1, int64_t bytes, int64_t rows, cudaStream_t s) {
    const cudaError_t e = cudaMemset2DAsync(dst, rows > 1 ? dst_nb1 : (size_t)bytes, 0, (size_t)bytes, (size_t)rows, s);
    if (e != cudaSuccess) return set_error(FB_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    return FB_OK;
}

}  // namespace

extern "C" {

int feml_b200_quantize_f8(int32_t xtype, const void *x, uint64_t x_nb1, int64_t rows, int64_t k, int64_t block_rows,
                          void *q, uint64_t q_nb1, float *scale, uint64_t scale_nb1, void *stream) {
    const char *op = "quantize_f8";
    FB_TRY(check_type(op, xtype));
    FB_TRY(check_dims(op, rows, k, 0));
    if (block_rows != 1 && block_rows != kB)
        return set_error(FB_ERR_UNSUPPORTED, "%s: blocks of %lld rows (1 or 128)", op, (long long)block_rows);
    if (rows == 0 || k == 0) return FB_OK;
    const fbk::F8Out o{q, stride_of(q_nb1, rows, k), scale, scale_nb1};
    FB_TRY(check_rows(op, "x", x, x_nb1, rows, k * esize(xtype), esize(xtype)));
    FB_TRY(check_out(op, o, rows, k, (rows + block_rows - 1) / block_rows));
    x_nb1 = stride_of(x_nb1, rows, k * esize(xtype));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (block_rows == 1) return fbk::launch_rows_f8(xtype, x, x_nb1, nullptr, 0, rows, k, o, s);
    return fbk::launch_quantize_f8_tiles(xtype, x, x_nb1, rows, k, o, s);
}

int feml_b200_rms_norm_f8(int32_t xtype, const void *x, uint64_t x_nb1, const void *residual, uint64_t residual_nb1,
                          void *sum, uint64_t sum_nb1, int32_t wtype, const void *weight, float eps, int64_t rows,
                          int64_t k, void *q, uint64_t q_nb1, float *scale, uint64_t scale_nb1, void *stream) {
    const char *op = "rms_norm_f8";
    FB_TRY(check_type(op, xtype));
    if (wtype != xtype && wtype != FB_F32)
        return set_error(FB_ERR_UNSUPPORTED, "%s: weight type %d (F32 or the type of x)", op, wtype);
    FB_TRY(check_dims(op, rows, k, 0));
    if (!(eps >= 0.0f)) return set_error(FB_ERR_INVALID, "%s: eps %g", op, (double)eps);
    if (rows == 0 || k == 0) return FB_OK;
    const int64_t es = esize(xtype);
    const fbk::F8Out o{q, stride_of(q_nb1, rows, k), scale, scale_nb1};
    FB_TRY(check_rows(op, "x", x, x_nb1, rows, k * es, es));
    FB_TRY(check_rows(op, "weight", weight, 0, 1, k * esize(wtype), esize(wtype)));
    if (residual) {
        FB_TRY(check_rows(op, "residual", residual, residual_nb1, rows, k * es, es));
        FB_TRY(check_rows(op, "sum", sum, sum_nb1, rows, k * es, es));
    }
    FB_TRY(check_out(op, o, rows, k, rows));
    return fbk::launch_rms_norm_f8(xtype, x, stride_of(x_nb1, rows, k * es), residual,
                                   stride_of(residual_nb1, rows, k * es), sum, stride_of(sum_nb1, rows, k * es), wtype,
                                   weight, eps, rows, k, o, static_cast<cudaStream_t>(stream));
}

int feml_b200_silu_mul_f8(int32_t xtype, const void *gate, uint64_t gate_nb1, const void *up, uint64_t up_nb1,
                          int64_t rows, int64_t k, void *q, uint64_t q_nb1, float *scale, uint64_t scale_nb1,
                          void *stream) {
    const char *op = "silu_mul_f8";
    FB_TRY(check_type(op, xtype));
    FB_TRY(check_dims(op, rows, k, 0));
    if (rows == 0 || k == 0) return FB_OK;
    const int64_t es = esize(xtype);
    const fbk::F8Out o{q, stride_of(q_nb1, rows, k), scale, scale_nb1};
    FB_TRY(check_rows(op, "gate", gate, gate_nb1, rows, k * es, es));
    FB_TRY(check_rows(op, "up", up, up_nb1, rows, k * es, es));
    FB_TRY(check_out(op, o, rows, k, rows));
    return fbk::launch_rows_f8(xtype, gate, stride_of(gate_nb1, rows, k * es), up, stride_of(up_nb1, rows, k * es), rows,
                               k, o, static_cast<cudaStream_t>(stream));
}

int feml_b200_mul_mat_f8(const void *w, uint64_t w_nb1, const float *w_scale, uint64_t w_scale_nb1, const void *x,
                         uint64_t x_nb1, const float *x_scale, uint64_t x_scale_nb1, int32_t dst_type, void *dst,
                         uint64_t dst_nb1, int64_t K, int64_t M, int64_t N, void *stream) {
    const char *op = "mul_mat_f8";
    FB_TRY(check_type(op, dst_type));
    FB_TRY(check_dims(op, K, M, N));
    if (M == 0 || N == 0) return FB_OK;
    const int64_t es = esize(dst_type), kb = (K + kB - 1) / kB;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    FB_TRY(check_rows(op, "dst", dst, dst_nb1, N, M * es, es));
    if (K == 0) return zero_rows(op, dst, dst_nb1, M * es, N, s);
    FB_TRY(check_rows(op, "w", w, w_nb1, M, K, 1));
    FB_TRY(check_rows(op, "w_scale", w_scale, w_scale_nb1, (M + kB - 1) / kB, kb * 4, 4));
    FB_TRY(check_rows(op, "x", x, x_nb1, N, K, 1));
    FB_TRY(check_rows(op, "x_scale", x_scale, x_scale_nb1, N, kb * 4, 4));
    fbk::F8Gemm p{};
    p.w = static_cast<const uint8_t *>(w);
    p.ws = reinterpret_cast<const uint8_t *>(w_scale);
    p.x = static_cast<const uint8_t *>(x);
    p.xs = reinterpret_cast<const uint8_t *>(x_scale);
    p.w_nb1 = stride_of(w_nb1, M, K);
    p.ws_nb1 = w_scale_nb1;
    p.x_nb1 = stride_of(x_nb1, N, K);
    p.xs_nb1 = x_scale_nb1;
    p.y = static_cast<uint8_t *>(dst);
    p.y_nb1 = stride_of(dst_nb1, N, M * es);
    p.out_type = dst_type;
    p.K = (int)K;
    p.M = (int)M;
    p.N = (int)N;
    return run_product(p, nullptr, 0, s);
}

int feml_b200_mul_mat_f8_plan(int64_t K, int64_t M, int64_t N, int64_t n_experts, int32_t *tile, int32_t *warps,
                              int64_t *ctas, int32_t *split) {
    const char *op = "mul_mat_f8_plan";
    if (!tile || !warps || !ctas || !split) return set_error(FB_ERR_INVALID, "%s: null out", op);
    FB_TRY(check_dims(op, K, M, N));
    if (n_experts < 0 || n_experts > kMaxF8Experts)
        return set_error(FB_ERR_UNSUPPORTED, "%s: %lld experts (0 to %lld)", op, (long long)n_experts, (long long)kMaxF8Experts);
    *tile = *warps = *split = 0;
    *ctas = 0;
    if (K == 0 || M == 0 || N == 0) return FB_OK;
    const fbk::F8Plan f = n_experts == 0 && N <= fbk::gemv_f8_max_rows() ? fbk::gemv_f8_plan(K, M)
                                                                         : fbk::gemm_f8_plan(K, M, N, n_experts);
    *tile = f.tile;
    *warps = f.warps;
    *ctas = f.ctas;
    *split = f.split;
    return FB_OK;
}

int feml_b200_mul_mat_f8_grouped_workspace(int64_t K, int64_t n_rows, int64_t n_experts, uint64_t *bytes) {
    const char *op = "mul_mat_f8_grouped_workspace";
    if (!bytes) return set_error(FB_ERR_INVALID, "%s: null out", op);
    *bytes = 0;
    FB_TRY(check_dims(op, K, n_rows, n_experts));
    if (fbk::gather_f8_pays(n_rows, n_experts)) *bytes = fbk::gather_f8_bytes(K, n_rows);
    return FB_OK;
}

int feml_b200_mul_mat_f8_grouped(const void *w, uint64_t w_nb1, uint64_t w_nb2, const float *w_scale,
                                 uint64_t w_scale_nb1, uint64_t w_scale_nb2, int64_t n_experts, const void *x,
                                 uint64_t x_nb1, int64_t n_x, const float *x_scale, uint64_t x_scale_nb1,
                                 const int32_t *counts, const int32_t *offsets, const int32_t *rows,
                                 int64_t n_selected, int32_t dst_type, void *dst, uint64_t dst_nb1, int64_t K,
                                 int64_t M, int64_t n_rows, void *workspace, uint64_t workspace_bytes, int32_t *status,
                                 void *stream) {
    const char *op = "mul_mat_f8_grouped";
    FB_TRY(check_type(op, dst_type));
    FB_TRY(check_dims(op, K, M, n_rows));
    FB_TRY(check_dims(op, n_x, n_selected, n_experts));
    if (n_experts < 1 || n_experts > kMaxF8Experts)
        return set_error(FB_ERR_UNSUPPORTED, "%s: %lld experts (1 to %lld)", op, (long long)n_experts, (long long)kMaxF8Experts);
    if (n_selected < 1) return set_error(FB_ERR_INVALID, "%s: n_selected %lld", op, (long long)n_selected);
    if (K == 0) return set_error(FB_ERR_UNSUPPORTED, "%s: K = 0", op);
    if (!rows && n_x < n_rows)
        return set_error(FB_ERR_SHAPE, "%s: %lld rows of x for %lld rows of dst", op, (long long)n_x, (long long)n_rows);
    if (M == 0 || n_rows == 0) return FB_OK;
    if (n_x == 0) return set_error(FB_ERR_SHAPE, "%s: x has no rows", op);
    const int64_t es = esize(dst_type), kb = (K + kB - 1) / kB, mb = (M + kB - 1) / kB;
    FB_TRY(check_rows(op, "dst", dst, dst_nb1, n_rows, M * es, es));
    FB_TRY(check_rows(op, "w", w, w_nb1, M, K, 1));
    FB_TRY(check_rows(op, "w_scale", w_scale, w_scale_nb1, mb, kb * 4, 4));
    FB_TRY(check_rows(op, "x", x, x_nb1, n_x, K, 1));
    FB_TRY(check_rows(op, "x_scale", x_scale, x_scale_nb1, n_x, kb * 4, 4));
    w_nb1 = stride_of(w_nb1, M, K);
    w_scale_nb1 = M > kB ? w_scale_nb1 : (uint64_t)(kb * 4);
    if (n_experts > 1 && w_scale_nb2 % 4) return set_error(FB_ERR_INVALID, "%s: w_scale is not aligned to its elements", op);
    FB_TRY(check_rows(op, "counts", counts, 0, 1, n_experts * 4, 4));
    FB_TRY(check_rows(op, "offsets", offsets, 0, 1, n_experts * 4, 4));
    if (rows) FB_TRY(check_rows(op, "rows", rows, 0, 1, n_rows * 4, 4));
    if (off(status, 0, 4)) return set_error(FB_ERR_INVALID, "%s: status is not 4-byte aligned", op);
    fbk::F8Gemm p{};
    p.w = static_cast<const uint8_t *>(w);
    p.ws = reinterpret_cast<const uint8_t *>(w_scale);
    p.x = static_cast<const uint8_t *>(x);
    p.xs = reinterpret_cast<const uint8_t *>(x_scale);
    p.w_nb1 = w_nb1;
    p.w_nb2 = n_experts > 1 ? w_nb2 : 0;
    p.ws_nb1 = w_scale_nb1;
    p.ws_nb2 = n_experts > 1 ? w_scale_nb2 : 0;
    p.x_nb1 = stride_of(x_nb1, n_x, K);
    p.xs_nb1 = x_scale_nb1;
    p.y = static_cast<uint8_t *>(dst);
    p.y_nb1 = stride_of(dst_nb1, n_rows, M * es);
    p.out_type = dst_type;
    p.K = (int)K;
    p.M = (int)M;
    p.N = (int)n_rows;
    p.g.counts = counts;
    p.g.offsets = offsets;
    p.g.rows = rows;
    p.g.n_experts = (int)n_experts;
    p.g.n_rows = (int)n_rows;
    p.g.n_selected = (int)n_selected;
    p.g.n_x = (int)n_x;
    p.status = status;
    return run_product(p, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
