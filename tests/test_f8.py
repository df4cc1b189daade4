"""Refusals of the e4m3 operators (no GPU): every argument check of the C
entry points comes before any device work, and the Python calls refuse what
is no CUDA tensor."""
import pytest
import torch

import feml_b200 as F
from feml_b200 import _lib, ops

F32, F16, BF16, P = 5, 4, 30, 4096  # P: an aligned address that is never touched
INVALID, UNSUPPORTED, SHAPE = 1, 2, 3


def call(name, *args):
    fn = getattr(_lib.lib(), "feml_b200_" + name)
    rc = fn(*args)
    if rc:
        assert name in _lib.lib().feml_b200_last_error().decode()
    return rc


def quantize(t=F32, x=P, x_nb1=512, rows=2, k=128, br=1, q=P, q_nb1=128, s=P, s_nb1=4):
    return call("quantize_f8", t, x, x_nb1, rows, k, br, q, q_nb1, s, s_nb1, 0)


def norm(t=BF16, x=P, x_nb1=256, r=P, r_nb1=256, h=P, h_nb1=256, wt=F32, w=P, eps=1e-5, rows=2, k=128, q=P, q_nb1=128,
         s=P, s_nb1=4):
    return call("rms_norm_f8", t, x, x_nb1, r, r_nb1, h, h_nb1, wt, w, eps, rows, k, q, q_nb1, s, s_nb1, 0)


def silu(t=F16, g=P, g_nb1=256, u=P, u_nb1=256, rows=2, k=128, q=P, q_nb1=128, s=P, s_nb1=4):
    return call("silu_mul_f8", t, g, g_nb1, u, u_nb1, rows, k, q, q_nb1, s, s_nb1, 0)


def mul_mat(w=P, w_nb1=256, ws=P, ws_nb1=8, x=P, x_nb1=256, xs=P, xs_nb1=8, t=F32, y=P, y_nb1=1200, K=256, M=300, N=2):
    return call("mul_mat_f8", w, w_nb1, ws, ws_nb1, x, x_nb1, xs, xs_nb1, t, y, y_nb1, K, M, N, 0)


def grouped(w=P, w_nb1=256, w_nb2=256 * 300, ws=P, ws_nb1=8, ws_nb2=24, E=4, x=P, x_nb1=256, n_x=2, xs=P, xs_nb1=8,
            counts=P, offsets=P, rows=P, sel=1, t=F32, y=P, y_nb1=1200, K=256, M=300, R=2, work=0, work_n=0, status=0):
    return call("mul_mat_f8_grouped", w, w_nb1, w_nb2, ws, ws_nb1, ws_nb2, E, x, x_nb1, n_x, xs, xs_nb1, counts, offsets,
                rows, sel, t, y, y_nb1, K, M, R, work, work_n, status, 0)


@pytest.mark.parametrize("fn,bad,code", [
    (quantize, dict(t=11), UNSUPPORTED), (quantize, dict(t=-1), UNSUPPORTED), (quantize, dict(rows=-1), INVALID),
    (quantize, dict(k=-1), INVALID), (quantize, dict(rows=1 << 31), UNSUPPORTED), (mul_mat, dict(K=2 ** 31 - 1), UNSUPPORTED), (quantize, dict(br=2), UNSUPPORTED),
    (quantize, dict(br=0), UNSUPPORTED), (quantize, dict(x=0), INVALID), (quantize, dict(q=0), INVALID),
    (quantize, dict(s=0), INVALID), (quantize, dict(x=P + 2), INVALID), (quantize, dict(x_nb1=514), INVALID),
    (quantize, dict(x_nb1=508), SHAPE), (quantize, dict(x_nb1=0), SHAPE), (quantize, dict(q_nb1=127), SHAPE),
    (quantize, dict(s_nb1=6), INVALID), (quantize, dict(s_nb1=0), SHAPE), (quantize, dict(k=129, x_nb1=516, q_nb1=129), SHAPE),
    (norm, dict(t=0), UNSUPPORTED), (norm, dict(wt=F16), UNSUPPORTED), (norm, dict(eps=-1.0), INVALID),
    (norm, dict(eps=float("nan")), INVALID), (norm, dict(x=0), INVALID), (norm, dict(w=0), INVALID), (norm, dict(h=0), INVALID),
    (norm, dict(w=P + 2), INVALID), (norm, dict(r_nb1=254), SHAPE), (norm, dict(h_nb1=128), SHAPE), (norm, dict(q=0), INVALID),
    (norm, dict(rows=-3), INVALID),
    (silu, dict(t=7), UNSUPPORTED), (silu, dict(g=0), INVALID), (silu, dict(u=0), INVALID), (silu, dict(u=P + 1), INVALID),
    (silu, dict(u_nb1=200), SHAPE), (silu, dict(s=P + 1), INVALID),
    (mul_mat, dict(t=11), UNSUPPORTED), (mul_mat, dict(K=-1), INVALID), (mul_mat, dict(M=-1), INVALID),
    (mul_mat, dict(N=-1), INVALID), (mul_mat, dict(N=1 << 31), UNSUPPORTED), (mul_mat, dict(w=0), INVALID),
    (mul_mat, dict(x=0), INVALID), (mul_mat, dict(ws=0), INVALID), (mul_mat, dict(xs=0), INVALID), (mul_mat, dict(y=0), INVALID),
    (mul_mat, dict(w_nb1=255), SHAPE), (mul_mat, dict(x_nb1=0), SHAPE), (mul_mat, dict(ws_nb1=4), SHAPE),
    (mul_mat, dict(xs_nb1=4), SHAPE), (mul_mat, dict(y_nb1=1196), SHAPE), (mul_mat, dict(y=P + 2), INVALID),
    (mul_mat, dict(xs=P + 2), INVALID), (mul_mat, dict(t=BF16, y=P + 1), INVALID),
    (grouped, dict(E=0), UNSUPPORTED), (grouped, dict(E=1025), UNSUPPORTED), (grouped, dict(sel=0), INVALID),
    (grouped, dict(K=0), UNSUPPORTED), (grouped, dict(rows=0, n_x=1), SHAPE), (grouped, dict(n_x=0), SHAPE),
    (grouped, dict(counts=0), INVALID), (grouped, dict(offsets=0), INVALID), (grouped, dict(offsets=P + 2), INVALID),
    (grouped, dict(rows=P + 2), INVALID), (grouped, dict(status=P + 2), INVALID), (grouped, dict(ws_nb2=26), INVALID),
    (grouped, dict(R=-1), INVALID), (grouped, dict(y=0), INVALID), (grouped, dict(w=0), INVALID),
])
def test_refusals(fn, bad, code):
    assert fn(**bad) == code


@pytest.mark.parametrize("fn,empty", [
    (quantize, dict(rows=0)), (quantize, dict(k=0)), (norm, dict(rows=0)), (silu, dict(k=0)), (mul_mat, dict(N=0)),
    (mul_mat, dict(M=0)), (grouped, dict(R=0)), (grouped, dict(M=0)),
])
def test_empty_operands_need_nothing(fn, empty):
    pointers = {quantize: ("x", "q", "s"), norm: ("x", "q", "s", "w"), silu: ("g", "u", "q", "s"),
                mul_mat: ("w", "x", "ws", "xs", "y"), grouped: ("w", "x", "ws", "xs", "y", "counts", "offsets", "rows")}[fn]
    assert fn(**empty, **{p: 0 for p in pointers if p not in empty}) == 0


def test_python_calls_refuse_host_tensors():
    x = torch.zeros(2, 128)
    q = torch.zeros(2, 128).to(torch.float8_e4m3fn)
    s = torch.zeros(2, 1)
    i = torch.zeros(1, dtype=torch.int32)
    for f in (lambda: ops.quantize_f8(x), lambda: ops.rms_norm_f8(x, x[0], 1e-5), lambda: ops.silu_mul_f8(x, x),
              lambda: ops.mul_mat_f8(q, s, q, s), lambda: ops.mul_mat_f8_grouped(q[None], s[None], q, s, i, i),
              lambda: ops.quantize_f8([1.0])):
        with pytest.raises(F.FemlError):
            f()


def test_product_plans():
    """The launch rules on the host (148 SMs without a GPU): rows per weight tile, warps, CTAs, CTAs per shared tile."""
    plan = ops.mul_mat_f8_plan
    assert plan(4096, 4096, 1) == (32, 16, 128, 1)      # one CTA of 16 warps per tile
    assert plan(4096, 14336, 16) == (32, 8, 448, 1)     # two of eight per SM and more
    assert plan(16384, 512, 8) == (32, 8, 128, 8)       # few tiles: clusters
    assert plan(14336, 4096, 64) == (128, 12, 128, 4)   # few row tiles: clusters
    assert plan(4096, 14336, 64) == (128, 12, 112, 1)
    assert plan(4096, 14336, 8192) == (256, 12, 148, 1)
    assert plan(4096, 14336, 16, 8) == (256, 12, 148, 1)
    assert plan(4096, 200, 20, 2) == (128, 12, 32, 8)
    assert plan(0, 5, 5) == plan(5, 0, 5) == plan(5, 5, 0) == (0, 0, 0, 0)
    for bad in ((-1, 1, 1, 0), (1, 2 ** 31, 1, 0), (1, 1, 1, -1), (1, 1, 1, 1025)):
        with pytest.raises(F.FemlError):
            plan(*bad)
