"""Kernel-level entry points of libfeml_b200.so on torch CUDA tensors.

torch only provides device memory and the current stream here; every op
runs a kernel of this library (include/feml_b200.h, section 3).
Layouts follow ggml: a weight matrix ne=[K, M] is a uint8 tensor [M, row_bytes];
activations ne=[K, N] are f32 [N, K]; results ne=[M, N] are f32 [N, M].
"""
import ctypes

import torch

from . import DType, FemlError, _check
from . import _lib as _L


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def row_bytes(dtype, k):
    return DType(dtype).row_size(k)


def quantize(dtype, x):
    """Quantize f32 rows [rows, k] -> uint8 [rows, row_bytes] (ggml blocks)."""
    assert x.is_cuda and x.dtype == torch.float32 and x.dim() == 2
    rows, k = x.shape
    out = torch.empty((rows, row_bytes(dtype, k)), dtype=torch.uint8, device=x.device)
    _check(_L.lib().feml_b200_quantize(int(dtype), _ptr(x), x.stride(0) * 4, _ptr(out), rows, k, _stream()))
    return out


def mul_mat_workspace(wtype, K, M, N):
    v = ctypes.c_uint64()
    _check(_L.lib().feml_b200_mul_mat_workspace(int(wtype), K, M, N, ctypes.byref(v)))
    return v.value


def mul_mat_launches(wtype, K, M, N):
    """Kernel launches one mul_mat of this shape enqueues."""
    v = ctypes.c_int32()
    _check(_L.lib().feml_b200_mul_mat_launches(int(wtype), K, M, N, ctypes.byref(v)))
    return v.value


def mul_mat(wtype, w, x, K, out=None, workspace=None):
    """w: uint8 [M, row_bytes] (or f32 [M, K] for F32); x: f32 [N, K] -> f32 [N, M]."""
    M = w.shape[0]
    N = x.shape[0]
    w_nb1 = w.stride(0) * w.element_size()
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=x.device)
    need = mul_mat_workspace(wtype, K, M, N)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws_ptr = _ptr(workspace) if workspace is not None else ctypes.c_void_p()
    ws_n = workspace.numel() if workspace is not None else 0
    _check(_L.lib().feml_b200_mul_mat(int(wtype), _ptr(w), w_nb1, _ptr(x), x.stride(0) * 4, _ptr(out),
                                      out.stride(0) * 4, K, M, N, ws_ptr, ws_n, _stream()))
    return out


def mul_mat_noalloc(wtype, w, x, K, out):
    """feml_b200_mul_mat_noalloc: mul_mat with the library's fixed device
    scratch (no workspace, no allocation inside the call); `out` is given."""
    M, N = w.shape[0], x.shape[0]
    _check(_L.lib().feml_b200_mul_mat_noalloc(int(wtype), _ptr(w), w.stride(0) * w.element_size(), _ptr(x),
                                              x.stride(0) * 4, _ptr(out), out.stride(0) * 4, K, M, N, _stream()))
    return out


def mul_mat_noalloc_limit():
    return int(_L.lib().feml_b200_mul_mat_noalloc_limit())


def mul_mat_id_workspace(wtype, K, M, N, n_selected, n_experts):
    v = ctypes.c_uint64()
    _check(_L.lib().feml_b200_mul_mat_id_workspace(int(wtype), K, M, N, n_selected, n_experts, ctypes.byref(v)))
    return v.value


def mul_mat_id(wtype, w, x, ids, K, out=None, workspace=None, status=None):
    """w: uint8 [E, M, row_bytes] (or f32 [E, M, K]); x: f32 [N, K];
    ids: int32 [N, n_sel] -> f32 [N, n_sel, M] (ggml dst ne=[M, n_sel, N])."""
    E, M = w.shape[0], w.shape[1]
    N, n_sel = ids.shape
    es = w.element_size()
    if out is None:
        out = torch.empty((N, n_sel, M), dtype=torch.float32, device=x.device)
    need = mul_mat_id_workspace(wtype, K, M, N, n_sel, E)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    _check(_L.lib().feml_b200_mul_mat_id(int(wtype), _ptr(w), w.stride(1) * es, w.stride(0) * es, E, _ptr(x),
                                         x.stride(0) * 4, _ptr(ids), ids.stride(0) * 4, n_sel, _ptr(out),
                                         out.stride(1) * 4, out.stride(0) * 4, K, M, N, _ptr(workspace),
                                         workspace.numel(), st, _stream()))
    return out


def local_experts(n_experts, shard, n_shards):
    """Experts owned by `shard` when expert e lives on shard e % n_shards."""
    return max(0, (n_experts - shard + n_shards - 1) // n_shards)


def mul_mat_id_shard(wtype, w_local, x, ids, K, n_experts, shard, n_shards, out, workspace=None, status=None):
    """Expert-sharded mul_mat_id: w_local holds the experts e with
    e % n_shards == shard (local index e // n_shards). Writes only the
    out[t, s, :] slots routed to those experts (invalid ids: zeros + status)."""
    E_loc, M = w_local.shape[0], w_local.shape[1]
    if E_loc != local_experts(n_experts, shard, n_shards):
        raise FemlError("msg", f"mul_mat_id_shard: shard {shard}/{n_shards} of {n_experts} experts holds "
                               f"{local_experts(n_experts, shard, n_shards)} experts, got {E_loc}")
    N, n_sel = ids.shape
    es = w_local.element_size()
    need = mul_mat_id_workspace(wtype, K, M, N, n_sel, max(E_loc, 1))
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    w_nb2 = w_local.stride(0) * es if E_loc > 0 else 0
    _check(_L.lib().feml_b200_mul_mat_id_shard(int(wtype), _ptr(w_local), w_local.stride(1) * es, w_nb2, n_experts,
                                               shard, n_shards, _ptr(x), x.stride(0) * 4, _ptr(ids),
                                               ids.stride(0) * 4, n_sel, _ptr(out), out.stride(1) * 4,
                                               out.stride(0) * 4, K, M, N, _ptr(workspace), workspace.numel(), st,
                                               _stream()))
    return out


def _ptr_array(ptrs):
    arr = (ctypes.c_void_p * len(ptrs))(*[ctypes.c_void_p(int(v)) for v in ptrs])
    return arr


def mul_mat_peer(wtype, w_local, x, K, dst0_ptrs, dst1_ptrs, flag_ptrs, dst_nb1, counter, epoch, status=None):
    """feml_b200_mul_mat_peer: this rank's rows of a row-sharded decode
    mul_mat stored straight into every rank's output buffer (raw device
    pointers, own memory or IPC mappings), then every rank's flag raised."""
    M, N = w_local.shape[0], x.shape[0]
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    n = len(flag_ptrs)
    _check(_L.lib().feml_b200_mul_mat_peer(int(wtype), _ptr(w_local), w_local.stride(0) * w_local.element_size(),
                                           _ptr(x), x.stride(0) * 4, _ptr_array(dst0_ptrs), _ptr_array(dst1_ptrs),
                                           _ptr_array(flag_ptrs), n, dst_nb1, _ptr(counter), _ptr(epoch), K, M, N, st,
                                           _stream()))


def mul_mat_id_peer(wtype, w_local, x, ids, K, n_experts, shard, n_shards, dst0_ptrs, dst1_ptrs, flag_ptrs,
                    dst_nb1, dst_nb2, M, counter, epoch, workspace, status=None, owner_tokens=0):
    """feml_b200_mul_mat_id_peer(_owned): this shard's experts of an
    expert-sharded mul_mat_id, every output slot stored straight into every
    rank's output buffer of this step (owner_tokens == 0) or only into the
    buffer of the rank that owns its token (token t on rank t // owner_tokens),
    then every rank's flag raised."""
    E_loc = w_local.shape[0]
    if E_loc != local_experts(n_experts, shard, n_shards):
        raise FemlError("msg", f"mul_mat_id_peer: shard {shard}/{n_shards} of {n_experts} experts holds "
                               f"{local_experts(n_experts, shard, n_shards)} experts, got {E_loc}")
    N, n_sel = ids.shape
    es = w_local.element_size()
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    _check(_L.lib().feml_b200_mul_mat_id_peer_owned(int(wtype), _ptr(w_local), w_local.stride(1) * es,
                                                    w_local.stride(0) * es, n_experts, shard, n_shards, _ptr(x),
                                                    x.stride(0) * 4, _ptr(ids), ids.stride(0) * 4, n_sel,
                                                    _ptr_array(dst0_ptrs), _ptr_array(dst1_ptrs),
                                                    _ptr_array(flag_ptrs), len(flag_ptrs), dst_nb1, dst_nb2,
                                                    int(owner_tokens), _ptr(counter), _ptr(epoch), K, M, N,
                                                    _ptr(workspace), workspace.numel(), st, _stream()))


def peer_wait(flag, epoch, n_ranks, status=None, timeout_us=None):
    """Enqueue the end of a fused step: wait for every rank's signal (bounded
    by `timeout_us`, default about a second; on expiry bit 0 of `status` is
    set and the stream continues)."""
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    if timeout_us is None:
        _check(_L.lib().feml_b200_peer_wait(_ptr(flag), _ptr(epoch), n_ranks, st, _stream()))
    else:
        _check(_L.lib().feml_b200_peer_wait_timeout(_ptr(flag), _ptr(epoch), n_ranks, int(timeout_us), st,
                                                    _stream()))


def moe_route(ids, n_experts, status=None):
    """ids int32 [N, n_sel] -> (counts, offsets, rows) int32 device tensors."""
    N, n_sel = ids.shape
    dev = ids.device
    counts = torch.zeros(n_experts, dtype=torch.int32, device=dev)
    offsets = torch.zeros(n_experts, dtype=torch.int32, device=dev)
    rows = torch.full((N * n_sel,), -1, dtype=torch.int32, device=dev)
    st = _ptr(status) if status is not None else ctypes.c_void_p()
    _check(_L.lib().feml_b200_moe_route(_ptr(ids), ids.stride(0) * 4, n_sel, N, n_experts, _ptr(counts),
                                        _ptr(offsets), _ptr(rows), st, _stream()))
    return counts, offsets, rows


def block_dots(wtype, w, xq, K):
    """Per-block int32 sums: w uint8 [M, row_bytes], xq uint8 [N, q8 row bytes]
    -> int32 [M, N, K/32]."""
    M, N = w.shape[0], xq.shape[0]
    out = torch.empty((M, N, K // 32), dtype=torch.int32, device=w.device)
    _check(_L.lib().feml_b200_block_dots(int(wtype), _ptr(w), w.stride(0), _ptr(xq), K, M, N, _ptr(out), _stream()))
    return out


# ---------------------------------------------------------------------------
# e4m3 operators (include/feml_b200.h, "e4m3 operators"): values are
# torch.float8_e4m3fn with one f32 scale per 128 values of a row
# (activations) or per 128 x 128 block (weights); a value is q * scale.
# ---------------------------------------------------------------------------
_F8 = torch.float8_e4m3fn
_F32 = torch.float32
_F8_TYPES = {torch.float32: 5, torch.float16: 4, torch.bfloat16: 30}

# A decode step is a handful of calls of a few microseconds each, so the
# checks below read each attribute once and the stream comes as a handle
# without a Stream object around it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _f8_refuse(op, name, t, dtype, shape, device):
    """The reason why `t` is not the operand that a call needs."""
    if not isinstance(t, torch.Tensor):
        raise FemlError("msg", f"{op}: {name} is not a tensor")
    if t.get_device() != device:
        raise FemlError("msg", f"{op}: {name} is on {t.device}, not on cuda:{device}")
    if t.dtype != dtype:
        raise FemlError("unsupported", f"{op}: {name} is {t.dtype}, not {dtype}")
    if tuple(t.shape) != shape:
        raise FemlError("shape", f"{op}: {name} is {list(t.shape)}, not {list(shape)}")
    raise FemlError("shape", f"{op}: the rows of {name} are not contiguous")


def _f8_check(op, name, t, dtype, shape, device):
    """The tensor of an operand: on CUDA device `device`, of `dtype` and
    `shape`, its last dimension contiguous. Returns its strides."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device:
        strides = t.stride()
        if not strides or strides[-1] == 1 or shape[-1] <= 1:
            return strides
    _f8_refuse(op, name, t, dtype, shape, device)


def _f8_input(op, name, x):
    """(type id, rows, k, row stride in bytes) of a 2D activation matrix."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise FemlError("msg", f"{op}: {name} is not a CUDA tensor")
    shape, strides = x.shape, x.stride()
    if len(shape) != 2:
        raise FemlError("shape", f"{op}: {name} is {list(shape)}, not 2-dimensional")
    tid = _F8_TYPES.get(x.dtype)
    if tid is None:
        raise FemlError("unsupported", f"{op}: {name} is {x.dtype} (float32, float16 and bfloat16)")
    if strides[1] != 1 and shape[1] > 1:
        raise FemlError("shape", f"{op}: the rows of {name} are not contiguous")
    return tid, shape[0], shape[1], strides[0] * (4 if tid == 5 else 2)


def _f8_out(op, out, scale, rows, k, block_rows, device):
    """The two outputs of a quantizing call, given or new, and the arguments
    that stand for them."""
    srows, kb = -(-rows // block_rows), -(-k // 128)
    if out is None:
        out = torch.empty((rows, k), dtype=_F8, device=f"cuda:{device}")
        nb1 = k
    else:
        nb1 = _f8_check(op, "out", out, _F8, (rows, k), device)[0]
    if scale is None:
        scale = torch.empty((srows, kb), dtype=_F32, device=f"cuda:{device}")
        scale_nb1 = kb * 4
    else:
        scale_nb1 = _f8_check(op, "scale", scale, _F32, (srows, kb), device)[0] * 4
    return out, scale, (out.data_ptr(), nb1, scale.data_ptr(), scale_nb1)


def _f8_call(device, fn, *args):
    """fn(*args, stream) on `device`'s current stream, with `device` current."""
    if device == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        _check(rc)


def quantize_f8(x, block_rows=1, out=None, scale=None):
    """x [rows, k] (f32, f16 or bf16) in the 8-bit form -> (q e4m3 [rows, k],
    scale f32 [ceil(rows / block_rows), ceil(k / 128)]): block_rows = 1 for
    activations, 128 for weights."""
    op = "quantize_f8"
    tid, rows, k, nb1 = _f8_input(op, "x", x)
    if block_rows not in (1, 128):
        raise FemlError("unsupported", f"{op}: blocks of {block_rows} rows (1 or 128)")
    dev = x.get_device()
    out, scale, o = _f8_out(op, out, scale, rows, k, block_rows, dev)
    _f8_call(dev, _L.lib().feml_b200_quantize_f8, tid, x.data_ptr(), nb1, rows, k, block_rows, *o)
    return out, scale


def rms_norm_f8(x, weight, eps, residual=None, residual_out=None, out=None, scale=None):
    """h = x + residual (rounded to x's type), h / sqrt(mean(h^2) + eps) *
    weight in the 8-bit form -> (q, scale, h); h is None without a residual.
    x, residual [rows, k]; weight [k] of x's type or f32. h is written to
    `residual_out`, which may be x or residual itself."""
    op = "rms_norm_f8"
    tid, rows, k, nb1 = _f8_input(op, "x", x)
    dev = x.get_device()
    wid = 5 if isinstance(weight, torch.Tensor) and weight.dtype is _F32 else tid
    _f8_check(op, "weight", weight, _F32 if wid == 5 else x.dtype, (k,), dev)
    r_ptr = r_nb1 = h_ptr = h_nb1 = 0
    if residual is not None:
        es = 4 if tid == 5 else 2
        r_nb1 = _f8_check(op, "residual", residual, x.dtype, (rows, k), dev)[0] * es
        if residual_out is None:
            residual_out = torch.empty((rows, k), dtype=x.dtype, device=x.device)
            h_nb1 = k * es
        else:
            h_nb1 = _f8_check(op, "residual_out", residual_out, x.dtype, (rows, k), dev)[0] * es
        r_ptr, h_ptr = residual.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise FemlError("msg", f"{op}: residual_out without a residual")
    out, scale, o = _f8_out(op, out, scale, rows, k, 1, dev)
    _f8_call(dev, _L.lib().feml_b200_rms_norm_f8, tid, x.data_ptr(), nb1, r_ptr, r_nb1, h_ptr, h_nb1, wid,
             weight.data_ptr(), eps, rows, k, *o)
    return out, scale, residual_out


def silu_mul_f8(gate, up, out=None, scale=None):
    """gate / (1 + exp(-gate)) * up in the 8-bit form -> (q, scale). gate and
    up [rows, k], for instance the two halves of one product's output."""
    op = "silu_mul_f8"
    tid, rows, k, nb1 = _f8_input(op, "gate", gate)
    dev = gate.get_device()
    up_nb1 = _f8_check(op, "up", up, gate.dtype, (rows, k), dev)[0] * (4 if tid == 5 else 2)
    out, scale, o = _f8_out(op, out, scale, rows, k, 1, dev)
    _f8_call(dev, _L.lib().feml_b200_silu_mul_f8, tid, gate.data_ptr(), nb1, up.data_ptr(), up_nb1, rows, k, *o)
    return out, scale


def _f8_dst(op, out, out_dtype, n, m, device):
    """Output of a product (f32 unless given), its type id and row stride in bytes."""
    if out is None:
        out = torch.empty((n, m), dtype=out_dtype or _F32, device=f"cuda:{device}")
    nb1 = _f8_check(op, "out", out, out_dtype or getattr(out, "dtype", None), (n, m), device)[0]
    tid = _F8_TYPES.get(out.dtype)
    if tid is None:
        raise FemlError("unsupported", f"{op}: out is {out.dtype} (float32, float16 and bfloat16)")
    return out, tid, nb1 * (4 if tid == 5 else 2)


def mul_mat_f8(w, w_scale, x, x_scale, out=None, out_dtype=None):
    """mul_mat on the 8-bit form: w e4m3 [M, K] with w_scale [ceil(M / 128),
    ceil(K / 128)], x e4m3 [N, K] with x_scale [N, ceil(K / 128)] -> [N, M]
    in f32 (or out_dtype: float16, bfloat16)."""
    op = "mul_mat_f8"
    if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dim() != 2:
        raise FemlError("msg", f"{op}: w is not a 2-dimensional CUDA tensor")
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise FemlError("msg", f"{op}: x is not a 2-dimensional tensor")
    dev = w.get_device()
    m, k = w.shape
    n, kb = x.shape[0], -(-k // 128)
    w_nb1 = _f8_check(op, "w", w, _F8, (m, k), dev)[0]
    ws_nb1 = _f8_check(op, "w_scale", w_scale, _F32, (-(-m // 128), kb), dev)[0] * 4
    x_nb1 = _f8_check(op, "x", x, _F8, (n, k), dev)[0]
    xs_nb1 = _f8_check(op, "x_scale", x_scale, _F32, (n, kb), dev)[0] * 4
    out, tid, nb1 = _f8_dst(op, out, out_dtype, n, m, dev)
    _f8_call(dev, _L.lib().feml_b200_mul_mat_f8, w.data_ptr(), w_nb1, w_scale.data_ptr(), ws_nb1, x.data_ptr(), x_nb1,
             x_scale.data_ptr(), xs_nb1, tid, out.data_ptr(), nb1, k, m, n)
    return out


def mul_mat_f8_plan(K, M, N, n_experts=0):
    """How a product of 16-byte aligned operands is cut -> (weight rows per
    tile, warps per CTA, CTAs, CTAs that share a tile): mul_mat_f8 of N rows,
    or with n_experts mul_mat_f8_grouped of N output rows."""
    tile, warps, ctas, split = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int64(), ctypes.c_int32()
    _check(_L.lib().feml_b200_mul_mat_f8_plan(K, M, N, n_experts, ctypes.byref(tile), ctypes.byref(warps),
                                              ctypes.byref(ctas), ctypes.byref(split)))
    return tile.value, warps.value, ctas.value, split.value


def mul_mat_f8_grouped_workspace(K, n_rows, n_experts):
    """Workspace bytes for a product of n_rows rows with a row table."""
    v = ctypes.c_uint64()
    _check(_L.lib().feml_b200_mul_mat_f8_grouped_workspace(K, n_rows, n_experts, ctypes.byref(v)))
    return v.value


def mul_mat_f8_grouped(w, w_scale, x, x_scale, counts, offsets, rows=None, n_selected=1, out=None, out_dtype=None,
                       workspace=None, status=None):
    """The product for rows grouped by expert: out[r] = expert e's weights
    times row rows[r] // n_selected of x (row r without `rows`), for r in
    [offsets[e], offsets[e] + counts[e]). w e4m3 [E, M, K], w_scale [E,
    ceil(M / 128), ceil(K / 128)], x e4m3 [n, K]; counts, offsets, rows:
    int32 as moe_route gives them. -> [len(rows) or n, M]; rows of `out` in no
    group are left as they were (zeros when `out` is not given). `workspace`:
    uint8, mul_mat_f8_grouped_workspace bytes (allocated when needed). `status`:
    int32 [1], bit 1 is set where a table points outside its range, bit 0 where
    a wait inside the kernel ran out (the rows concerned are NaN)."""
    op = "mul_mat_f8_grouped"
    if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dim() != 3:
        raise FemlError("msg", f"{op}: w is not a 3-dimensional CUDA tensor")
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise FemlError("msg", f"{op}: x is not a 2-dimensional tensor")
    dev = w.get_device()
    e, m, k = w.shape
    n, kb = x.shape[0], -(-k // 128)
    w_nb2, w_nb1, _ = _f8_check(op, "w", w, _F8, (e, m, k), dev)
    ws_nb2, ws_nb1, _ = _f8_check(op, "w_scale", w_scale, _F32, (e, -(-m // 128), kb), dev)
    x_nb1 = _f8_check(op, "x", x, _F8, (n, k), dev)[0]
    xs_nb1 = _f8_check(op, "x_scale", x_scale, _F32, (n, kb), dev)[0]
    _f8_check(op, "counts", counts, torch.int32, (e,), dev)
    _f8_check(op, "offsets", offsets, torch.int32, (e,), dev)
    n_rows = n
    if rows is not None:
        n_rows = rows.numel() if isinstance(rows, torch.Tensor) else 0
        _f8_check(op, "rows", rows, torch.int32, (n_rows,), dev)
        if workspace is None:
            need = mul_mat_f8_grouped_workspace(k, n_rows, e)
            if need:
                workspace = torch.empty(need, dtype=torch.uint8, device=w.device)
    elif n_selected != 1:
        raise FemlError("msg", f"{op}: n_selected = {n_selected} without rows")
    if workspace is not None:
        _f8_check(op, "workspace", workspace, torch.uint8, (workspace.numel() if isinstance(workspace, torch.Tensor) else 0,), dev)
    if status is not None:
        _f8_check(op, "status", status, torch.int32, (1,), dev)
    if out is None:
        out = torch.zeros((n_rows, m), dtype=out_dtype or _F32, device=w.device)
    out, tid, nb1 = _f8_dst(op, out, out_dtype, n_rows, m, dev)
    _f8_call(dev, _L.lib().feml_b200_mul_mat_f8_grouped, w.data_ptr(), w_nb1, w_nb2, w_scale.data_ptr(), ws_nb1 * 4,
             ws_nb2 * 4, e, x.data_ptr(), x_nb1, n, x_scale.data_ptr(), xs_nb1 * 4, counts.data_ptr(),
             offsets.data_ptr(), rows.data_ptr() if rows is not None else 0, int(n_selected), tid, out.data_ptr(), nb1, k, m,
             n_rows, workspace.data_ptr() if workspace is not None else 0,
             workspace.numel() if workspace is not None else 0, status.data_ptr() if status is not None else 0)
    return out


__all__ = ["quantize", "mul_mat", "mul_mat_launches", "mul_mat_workspace", "mul_mat_noalloc", "mul_mat_noalloc_limit", "mul_mat_id", "mul_mat_id_workspace", "mul_mat_id_shard",
           "local_experts", "mul_mat_peer", "mul_mat_id_peer", "peer_wait", "moe_route",
           "block_dots", "row_bytes", "quantize_f8", "rms_norm_f8", "silu_mul_f8", "mul_mat_f8", "mul_mat_f8_plan", "mul_mat_f8_grouped", "mul_mat_f8_grouped_workspace", "FemlError"]
