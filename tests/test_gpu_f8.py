"""The e4m3 operators on the GPU against the same formulas in 64 bits.

Tolerances (u = 2^-24, the half step of f32):
  scales    a / 448: one division, plus the error of the largest value itself
  q         half a step of e4m3 around the exact value: 2^-4 of it, 2^-10
            below the normal range, both widened by the value's f32 error
  products  every f32 addition is off by at most 2u of the running sum of
            magnitudes (the tensor core may cut instead of rounding):
            A * 2u * (128 + blocks + 4), A = sum |x w| with scales, and half
            a step of the output type
"""
import math

import numpy as np
import pytest
import torch

import feml_b200 as F
from feml_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F8 = torch.float8_e4m3fn
FLOOR = 2.0 ** -100


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def blocks64(y, rows):
    """Exact (q before rounding, scale) of a 64-bit matrix."""
    r, k = y.shape
    pad = torch.nn.functional.pad(y, (0, -k % 128, 0, -r % rows))
    b = pad.reshape(pad.shape[0] // rows, rows, pad.shape[1] // 128, 128)
    scale = b.abs().amax((1, 3)).clamp_min(FLOOR) / 448
    q = (b / scale[:, None, :, None]).reshape(pad.shape)[:r, :k]
    return q, scale


def check_f8(q, s, y, rows=1, rel=0.0):
    """q, s against the 64-bit values y; rel: how far an f32 value of y may be off before it is quantized. A whole
    block's factor carries the error of its largest value, so q's value is off by 2 * rel and three roundings."""
    wq, ws = blocks64(y, rows)
    assert q.dtype == F8 and s.dtype == torch.float32
    assert torch.all((s.double() - ws).abs() <= ws * (rel + 2 * U))
    got = q.double()
    assert torch.isfinite(got).all()
    slack = 1 + 2 * rel + 4 * U
    step = torch.clamp(wq.abs() * 2.0 ** -4, min=2.0 ** -10)
    assert torch.all((got - wq).abs() <= step * slack + wq.abs() * (slack - 1)), float(((got - wq).abs() - step).max())


def to_f8(x, rows):
    """An f32 matrix in the 8-bit form, by torch."""
    q, s = blocks64(x.double(), rows)
    return q.float().clamp(-448, 448).to(F8), s.float()


def product64(w, ws, x, xs):
    """Exact product and the sum of magnitudes."""
    k = torch.arange(w.shape[1], device="cuda") // 128
    m = torch.arange(w.shape[0], device="cuda") // 128
    a = x.double() * xs.double()[:, k]
    b = w.double() * ws.double()[m][:, k]
    return a @ b.T, a.abs() @ b.abs().T


def check_product(got, want, mags, K):
    tol = mags * (2 * U) * (128 + -(-K // 128) + 4) + want.abs() * HALF[got.dtype] * (1 + 2.0 ** -10)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half the smallest f16
    err = (got.double() - want).abs()
    assert torch.all(err <= tol), (float((err - tol).max()), float(err.max()))


# ---------------------------------------------------------------------------------------------------------------
# row operators
# ---------------------------------------------------------------------------------------------------------------
ROWS = [(1, 128), (1, 1), (3, 127), (5, 129), (1, 4096), (2, 4100), (7, 1000), (33, 8), (130, 384), (1, 16384), (300, 2048)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,k", ROWS + [(128, 128), (129, 257), (1000, 200)])
def test_quantize(t, block_rows, rows, k):
    x = rand(gen(rows * 7 + k), rows, k, scale=3.0).to(t)
    q, s = ops.quantize_f8(x, block_rows)
    check_f8(q, s, x.double(), block_rows)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("pad,lead", [(8, 0), (1, 0), (0, 1), (24, 8), (3, 5)])
def test_quantize_strides(t, block_rows, pad, lead):
    """Rows inside a wider matrix, starting at any element; outputs into wider buffers whose rest is kept."""
    rows, k = 131, 272
    x = rand(gen(pad + lead), rows, lead + k + pad).to(t)[:, lead:lead + k]
    out = torch.full((rows, k + pad + lead), 1.5, device="cuda").to(F8)
    scale = torch.full((-(-rows // block_rows), 3 + pad), 7.0, device="cuda")
    q, s = ops.quantize_f8(x, block_rows, out=out[:, lead:lead + k], scale=scale[:, :3])
    check_f8(q, s, x.double(), block_rows)
    want = torch.empty((rows, k), dtype=F8, device="cuda")
    ops.quantize_f8(x.contiguous(), block_rows, out=want)
    assert torch.equal(q.contiguous().view(torch.uint8), want.view(torch.uint8))
    assert torch.all(out[:, :lead].float() == 1.5) and torch.all(out[:, lead + k:].float() == 1.5)
    assert torch.all(scale[:, 3:] == 7.0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("k", [512, 515])
def test_quantize_special_values(t, block_rows, k):
    """Zero blocks, the smallest values of the type, infinities and NaN: a block with one of the last two is NaN
    throughout, its neighbours are not touched by it."""
    x = rand(gen(3), 256, k).to(t)
    x[0:128, 0:128] = 0
    x[0:128, 128:256] = torch.finfo(t).smallest_normal
    x[5, 256 + 17] = math.inf
    x[6, 384 + 100] = math.nan
    x[7, 384 + 3] = -math.inf
    x[128:256, 0:128] = -torch.finfo(t).max
    q, s = ops.quantize_f8(x, block_rows)
    bad = ~torch.isfinite(x.double())
    _, ws = blocks64(x.double().nan_to_num(0, 0, 0), block_rows)
    ref = torch.nn.functional.pad(bad, (0, -k % 128, 0, -256 % block_rows))
    ref = ref.reshape(256 // block_rows, block_rows, -1, 128).any(3).any(1)
    assert torch.equal(torch.isnan(s), ref)
    assert torch.all((s.double() - ws).abs()[~ref] <= ws[~ref] * 2 * U)
    spread = ref.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:256, :k]
    assert torch.equal(torch.isnan(q.float()), spread)
    assert torch.all(q.float()[0:128, 0:128] == 0)
    assert torch.all(q.float()[128:256, 0:128] == -448)


def test_scale_and_factor_are_correctly_rounded():
    """scale = a / 448 and the factor 448 / a as IEEE division gives them: every mantissa of a, and a part of them at
    every exponent that a block maximum can have. The factor shows through two neighbouring values of each row: the
    last whose product with it is at most 17, halfway between the e4m3 values 16 and 18 (to even: 16), and the next."""
    f = np.float32
    m = (np.arange(1 << 23, dtype=np.uint32) | np.uint32(0x3F800000)).view(f)
    r = f(448) / m
    y = f(17) / r
    for _ in range(4):
        y = np.where(y * r > f(17), np.nextafter(y, f(0)), y)
    for _ in range(4):
        up = np.nextafter(y, f(1))
        y = np.where(up * r <= f(17), up, y)
    up = np.nextafter(y, f(1))
    assert np.all(y * r <= f(17)) and np.all(up * r > f(17))
    x = np.stack([m, y, up], 1)
    s = m / f(448)
    q = torch.tensor([448.0, 16.0, 18.0], device="cuda").to(F8).view(torch.uint8)

    def same(x, s):
        got, scale = ops.quantize_f8(torch.from_numpy(x).cuda())
        assert torch.equal(scale[:, 0], torch.from_numpy(s).cuda())
        assert torch.equal(got.view(torch.uint8), q.expand(len(x), 3))

    same(x, s)
    part = np.random.default_rng(1).integers(0, 1 << 23, 1 << 12)
    for e in range(-100, 128):
        same(np.ldexp(x[part], e), np.ldexp(s[part], e))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("wt", ["same", "f32"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k", ROWS + [(1500, 512), (1025, 1000), (400, 4096), (2, 32768), (2, 70000), (3, 33000)])
def test_rms_norm(t, wt, residual, rows, k):
    g = gen(rows + k)
    x = rand(g, rows, k, scale=2.0).to(t)
    r = rand(g, rows, k, scale=5.0).to(t) if residual else None
    w = (1 + 0.2 * rand(g, k)).to(torch.float32 if wt == "f32" else t)
    q, s, h = ops.rms_norm_f8(x, w, 1e-5, residual=r)
    if residual:
        assert torch.equal(h, (x.float() + r.float()).to(t))
        base = h.double()
    else:
        assert h is None
        base = x.double()
    y = base / torch.sqrt((base * base).mean(1, keepdim=True) + 1e-5) * w.double()
    # longest chain of f32 additions of the sum of squares: 96; half of it after the square root; four more roundings
    check_f8(q, s, y, rel=(48 + 4) * U)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("into", ["x", "residual", "strided"])
@pytest.mark.parametrize("k", [1024, 1001, 66000])
def test_rms_norm_sum_in_place(t, into, k):
    g = gen(k)
    wide = rand(g, 9, 2 * k).to(t)
    x, r = (wide[:, :k], wide[:, k:]) if into == "strided" else (wide[:, :k].contiguous(), wide[:, k:].contiguous())
    want_h = (x.float() + r.float()).to(t)
    w = 1 + 0.1 * rand(g, k)
    q0, s0, h0 = ops.rms_norm_f8(x, w, 1e-6, residual=r)
    q1, s1, h1 = ops.rms_norm_f8(x, w, 1e-6, residual=r, residual_out=x if into == "x" else r)
    assert h1 is (x if into == "x" else r)
    assert torch.equal(h0, want_h) and torch.equal(h1, want_h)
    assert torch.equal(s0, s1) and torch.equal(q0.view(torch.uint8), q1.view(torch.uint8))
    # the fused call gives the bits of the two steps
    q2, s2, _ = ops.rms_norm_f8(want_h, w, 1e-6)
    assert torch.equal(s0, s2) and torch.equal(q0.view(torch.uint8), q2.view(torch.uint8))


def test_rms_norm_zero_and_broken_rows():
    x = torch.randn(6, 512, device="cuda")
    x[1] = 0
    x[2, 300] = math.nan
    x[3, 5] = math.inf
    q, s, _ = ops.rms_norm_f8(x, torch.ones(512, device="cuda"), 1e-5)
    assert torch.all(q[1].float() == 0) and torch.isfinite(s[1]).all()
    assert torch.isnan(s[2]).all() and torch.isnan(q[2].float()).all()
    assert torch.isnan(s[3, 0]) and torch.isnan(q[3, :128].float()).all()  # inf * 0; the rest of the row is 0
    assert torch.all(q[3, 128:].float() == 0)
    assert torch.isfinite(s[4:]).all() and torch.isfinite(q[4:].float()).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k", ROWS)
def test_silu_mul(t, rows, k):
    both = rand(gen(k + rows), rows, 2 * k, scale=4.0).clamp(-20, 20).to(t)
    gate, up = both[:, :k], both[:, k:]
    q, s = ops.silu_mul_f8(gate, up)
    g = gate.double()
    y = g / (1 + torch.exp(-g)) * up.double()
    # the fast exponential is off by up to 2 + 1.173 * 20 units of 2^-23, the division by 2, two products
    check_f8(q, s, y, rel=2 * U * (2 + 1.173 * 20 + 2 + 2))


def test_silu_mul_far_gates():
    gate = torch.tensor([[-200.0, -90.0, 0.0, 90.0, 200.0, 3e38, -3e38] + [1.0] * 121], device="cuda")
    up = torch.ones_like(gate)
    up[0, 5] = 1e-36
    q, s = ops.silu_mul_f8(gate, up)
    want = gate.double() * torch.sigmoid(gate.double()) * up.double()
    check_f8(q, s, want, rel=64 * U)


def test_silu_mul_subnormal_sigmoid():
    """1 / (1 + exp(-gate)) is below the normal f32 range, the product with a large `up` is not."""
    gate = torch.tensor([[-88.5, -88.0, -87.75, -87.5, -87.25, -87.0, -80.0, -60.0] * 16], device="cuda")
    up = torch.full_like(gate, 3e38)
    q, s = ops.silu_mul_f8(gate, up)
    g = gate.double()
    # the exponential as above; the reciprocal 2^-127 and below has 22 bits left, one unit of which is 2^-22
    check_f8(q, s, g / (1 + torch.exp(-g)) * up.double(), rel=2 * U * (2 + 1.173 * 88.5 + 2 + 2 + 2))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("u", [3e38, -1e30, 1.0])
@pytest.mark.parametrize("k", [1, 128, 136, 131])
def test_silu_mul_gates_past_the_exponential(t, u, k):
    """exp(-gate) is infinite in f32 below -88.7; the product with a large `up` is not 0 there. Every gate has blocks
    of its own (single elements, 32-byte vectors, 16-byte ones), so their scales show it to f32's precision."""
    gate = torch.cat([torch.linspace(-92.0, -86.0, 193), torch.linspace(-180.0, 0.0, 181)]).to(t).cuda()[:, None]
    gate = gate.repeat(1, k)
    up = torch.full_like(gate, u)
    q, s = ops.silu_mul_f8(gate, up)
    g = gate.double()
    y = g * torch.exp(g) / (1 + torch.exp(g)) * up.double()
    # each factor e^(g/2) is off by up to 2 + 1.173 * |g| / 2 units of 2^-23, the reciprocal by 1; four products, a sum
    wq, ws = blocks64(y, 1)
    rel = 2 * U * (4 + 1.173 * g[:, :1].abs() + 1 + 2 + 0.5)
    assert torch.all((s.double() - ws).abs() <= ws * (rel + 2 * U))
    check_f8(q, s, y, rel=2 * U * (4 + 1.173 * 180 + 3.5))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [512, 515])
def test_silu_mul_far_gates_among_near_ones(t, k):
    """A lane with one far gate computes its near ones as the other lanes do, up to the last bits."""
    g = gen(k)
    gate = rand(g, 40, k, scale=2.0).to(t)
    gate[::3, 7::31] = torch.tensor([-87.0, -87.5, -100.0, -500.0]).to(t).cuda().repeat(1, 99)[0, :gate[0, 7::31].numel()]
    up = rand(g, 40, k, scale=3.0).to(t)
    q, s = ops.silu_mul_f8(gate, up)
    d = gate.double()
    check_f8(q, s, d * torch.sigmoid(d) * up.double(), rel=2 * U * (4 + 1.173 * 20 + 3.5))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_silu_mul_subnormal_gates(t):
    """A gate below the normal range keeps its bits (f32 and bf16 have the same exponents)."""
    least = 2.0 ** -149 if t == torch.float32 else 2.0 ** -133
    gate = (torch.tensor([1.0, 3.0, 5.0, 127.0, -1.0, -7.0], dtype=torch.float64) * least).to(t).cuda()[:, None]
    up = torch.full_like(gate, 2.0 ** 127)
    q, s = ops.silu_mul_f8(gate, up)
    # the reciprocal of 2 is off by one unit at most; two products that are not exact powers of two
    check_f8(q, s, gate.double() / 2 * up.double(), rel=2 * U * 3)


# ---------------------------------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------------------------------
def operands(seed, n, k, m, e=None):
    g = gen(seed)
    x, xs = to_f8(rand(g, n, k) * torch.exp(rand(g, n, 1)), 1)
    if e is None:
        w, ws = to_f8(rand(g, m, k, scale=0.05), 128)
        return w, ws, x, xs
    ws, qs = [], []
    for _ in range(e):
        q, s = to_f8(rand(g, m, k, scale=0.05), 128)
        qs.append(q)
        ws.append(s)
    return torch.stack(qs), torch.stack(ws), x, xs


SHAPES = [(1, 128, 128), (1, 4096, 512), (1, 16, 1), (2, 144, 130), (3, 4096, 1000), (8, 1024, 64), (9, 512, 129),
          (16, 2048, 300), (17, 1040, 257), (33, 640, 384), (64, 2048, 200), (65, 256, 513), (128, 1152, 256),
          (129, 384, 640), (200, 4112, 129), (256, 512, 1000), (300, 2048, 2300), (513, 272, 1025), (1030, 1536, 700)]
ODD = [(1, 1, 1), (1, 127, 5), (3, 129, 130), (40, 1001, 65), (130, 300, 70), (2, 4099, 33)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", SHAPES + ODD)
def test_mul_mat(t, n, k, m):
    w, ws, x, xs = operands(n + k + m, n, k, m)
    got = ops.mul_mat_f8(w, ws, x, xs, out_dtype=t)
    assert got.dtype == t
    check_product(got, *product64(w, ws, x, xs), k)


@pytest.mark.parametrize("n", [1, 5, 20, 150])
@pytest.mark.parametrize("wpad,xpad,ypad", [(16, 0, 0), (0, 32, 4), (16, 16, 1), (1, 0, 3), (0, 5, 0), (3, 7, 8)])
def test_mul_mat_strides(n, wpad, xpad, ypad):
    """Operands inside wider matrices; the rest of the output buffer is kept."""
    k, m = 400, 270
    w, ws, x, xs = operands(n, n, k + max(wpad, xpad), m)
    w, x = w.view(torch.uint8), x.view(torch.uint8)
    wv = torch.nn.functional.pad(w[:, :k], (0, wpad)).view(F8)[:, :k]
    xv = torch.nn.functional.pad(x[:, :k], (0, xpad)).view(F8)[:, :k]
    wsv, xsv = ws[:, :4], xs[:, :4]  # (strided where the pad adds a block)
    for t in (torch.float32, torch.bfloat16):
        out = torch.full((n, m + ypad), 3.0, dtype=t, device="cuda")
        got = ops.mul_mat_f8(wv, wsv, xv, xsv, out=out[:, :m])
        check_product(got, *product64(wv, wsv, xv, xsv), k)
        assert torch.all(out[:, m:] == 3.0)


@pytest.mark.parametrize("n", [2, 30, 200])
def test_mul_mat_offset_pointers(n):
    """Operands whose first element is on any byte."""
    k, m = 256, 140
    w, ws, x, xs = operands(n + 50, n, k, m)
    for off in (1, 2, 4, 8):
        wb = torch.zeros(m * k + off, dtype=torch.uint8, device="cuda")
        wb[off:] = w.view(torch.uint8).flatten()
        got = ops.mul_mat_f8(wb[off:].view(F8).view(m, k), ws, x, xs)
        check_product(got, *product64(w, ws, x, xs), k)
        ob = torch.full((n * m + off,), 9.0, dtype=torch.bfloat16, device="cuda")
        got = ops.mul_mat_f8(w, ws, x, xs, out=ob[off:].view(n, m))
        check_product(got, *product64(w, ws, x, xs), k)
        assert torch.all(ob[:off] == 9.0)


@pytest.mark.parametrize("m", [65535 * 64, 65535 * 64 + 1, 65535 * 64 * 2 + 70])
def test_mul_mat_many_rows_of_any_alignment(m):
    """More tiles of weight rows than one dimension of a grid has."""
    w, ws, x, xs = operands(m % 1000, 2, 1, 300)
    w = torch.cat([w.view(torch.uint8)] * (m // 300) + [w.view(torch.uint8)[:m % 300]]).view(F8)
    ws = torch.rand(-(-m // 128), 1, generator=gen(1), device="cuda") + 0.5
    buf = torch.full((2, m + 3), 5.0, dtype=torch.float16, device="cuda")
    got = ops.mul_mat_f8(w, ws, x, xs, out=buf[:, :m])
    check_product(got, *product64(w, ws, x, xs), 1)
    assert torch.all(buf[:, m:] == 5.0)


@pytest.mark.parametrize("n", [1, 12, 40, 140])
def test_mul_mat_nan_and_range(n):
    """A NaN value or scale reaches its own rows and columns and no others; extreme scales keep their range."""
    k, m = 512, 300
    w, ws, x, xs = operands(n + 9, n, k, m)
    xb = x.view(torch.uint8).clone()
    xb[0, 130] = 0x7F
    wb = w.view(torch.uint8).clone()
    wb[7, 3] = 0xFF
    got = ops.mul_mat_f8(wb.view(F8), ws, xb.view(F8), xs)
    want = torch.zeros_like(got, dtype=torch.bool)
    want[0] = True
    want[:, 7] = True
    assert torch.equal(torch.isnan(got), want)
    ws2 = ws.clone()
    ws2[2, 1] = math.nan  # weight rows 256..299
    got = ops.mul_mat_f8(w, ws2, x, xs)
    assert torch.isnan(got[:, 256:]).all() and torch.isfinite(got[:, :256]).all()
    big = ops.mul_mat_f8(w, ws * 2.0 ** 60, x, xs * 2.0 ** -60)
    assert torch.equal(big, ops.mul_mat_f8(w, ws, x, xs))


@pytest.mark.parametrize("n", [1, 4, 16, 33, 100, 260])
def test_mul_mat_is_deterministic_and_row_wise(n):
    """The same bits every time."""
    w, ws, x, xs = operands(n, n, 2048, 520)
    a = ops.mul_mat_f8(w, ws, x, xs)
    for _ in range(3):
        assert torch.equal(a, ops.mul_mat_f8(w, ws, x, xs))


def test_mul_mat_empty_sum():
    w = torch.empty(5, 0, dtype=F8, device="cuda")
    x = torch.empty(3, 0, dtype=F8, device="cuda")
    z = torch.empty(1, 0, device="cuda")
    out = torch.full((3, 9), 2.0, device="cuda")
    got = ops.mul_mat_f8(w, z, x, torch.empty(3, 0, device="cuda"), out=out[:, :5])
    assert torch.all(got == 0) and torch.all(out[:, 5:] == 2.0)


# ---------------------------------------------------------------------------------------------------------------
# groups
# ---------------------------------------------------------------------------------------------------------------
def tables(counts, gap=0):
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    o = (torch.cumsum(c, 0) - c).to(torch.int32) + gap
    return c, o


def check_grouped(got, w, ws, x, xs, counts, offsets, source, K):
    for e, (c, o) in enumerate(zip(counts, offsets)):
        if c:
            rows = source[o:o + c]
            check_product(got[o:o + c], *product64(w[e], ws[e], x[rows], xs[rows]), K)


GROUPS = [[1], [0], [5, 0, 3], [1, 1, 1, 1], [0, 0, 7], [130, 2, 0, 64], [128, 128], [33, 257, 1, 0, 12], [300]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("counts", GROUPS)
@pytest.mark.parametrize("k,m", [(256, 128), (528, 300), (129, 70)])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(t, counts, k, m, gather):
    """Ragged and empty groups, with rows before, between and behind them that are kept."""
    e, total, gap = len(counts), sum(counts), 3
    c, o = tables(counts, gap)
    n_rows = total + gap + 6
    n = 37 if gather else n_rows
    w, ws, x, xs = operands(k + total, n, k, m, e)
    g = gen(total)
    rows = torch.randint(0, 2 * n, (n_rows,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    source = (rows // 2).long() if gather else torch.arange(n_rows, device="cuda")
    out = torch.full((n_rows, m), 5.0, dtype=t, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, n_selected=2 if gather else 1, out=out, status=status)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), source, k)
    assert torch.all(got[:gap] == 5.0) and torch.all(got[gap + total:] == 5.0)
    assert int(status) == 0


@pytest.mark.parametrize("room", ["none", "short", "odd", "right"])
def test_grouped_workspace(room):
    """With any workspace, or none that can be used, the same bits; rows behind the groups may hold any index."""
    e, k, m, n = 2, 272, 130, 50
    counts = [70, 41]
    c, o = tables(counts)
    w, ws, x, xs = operands(3, n, k, m, e)
    rows = torch.randint(0, 3 * n, (120,), generator=gen(9), device="cuda", dtype=torch.int32)
    rows[111:] = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, 3 * n, 0, 1, 2, 3, 4], dtype=torch.int32, device="cuda")
    need = ops.mul_mat_f8_grouped_workspace(k, 120, e)
    assert need > 0 and ops.mul_mat_f8_grouped_workspace(k, 16 * e, e) == 0
    work = {"none": torch.empty(0, dtype=torch.uint8, device="cuda"), "short": torch.empty(need - 1, dtype=torch.uint8, device="cuda"),
            "odd": torch.empty(need + 1, dtype=torch.uint8, device="cuda")[1:], "right": torch.empty(need, dtype=torch.uint8, device="cuda")}
    out = torch.full((120, m), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, n_selected=3, out=out, workspace=work[room], status=status)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), (rows // 3).long(), k)
    assert torch.all(got[111:] == 5.0) and int(status) == 0
    assert torch.equal(got[:111], ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, n_selected=3)[:111])


def test_grouped_many_experts():
    e, k, m = 300, 128, 48
    g = gen(1)
    counts = torch.randint(0, 4, (e,), generator=g, device="cuda").tolist()
    counts[17] = 150
    c, o = tables(counts)
    n = sum(counts)
    w, ws, x, xs = operands(4, n, k, m, e)
    got = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), torch.arange(n, device="cuda"), k)


@pytest.mark.parametrize("k", [256, 131])
def test_grouped_strides(k):
    """Experts and rows inside wider tensors, experts in another order of dimensions, one expert's weights for all."""
    e, m, counts = 3, 150, [20, 0, 70]
    c, o = tables(counts)
    w, ws, x, xs = operands(8, 90, k, m, e)
    src = torch.arange(90, device="cuda")
    wide = torch.zeros(e, m + 2, k + 16, dtype=torch.uint8, device="cuda")
    wide[:, :m, :k] = w.view(torch.uint8)
    wide_s = torch.zeros(e, 4, 5, device="cuda")
    wide_s[:, :2, :ws.shape[2]] = ws
    got = ops.mul_mat_f8_grouped(wide.view(F8)[:, :m, :k], wide_s[:, :2, :ws.shape[2]], x, xs, c, o)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), src, k)
    inner = w.view(torch.uint8).permute(1, 0, 2).contiguous().view(F8).permute(1, 0, 2)
    got = ops.mul_mat_f8_grouped(inner, ws, x, xs, c, o)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), src, k)
    one = w[:1].expand(e, m, k)
    got = ops.mul_mat_f8_grouped(one, ws[:1].expand(e, -1, -1), x, xs, c, o)
    check_grouped(got, one, ws[:1].expand(e, -1, -1), x, xs, counts, o.tolist(), src, k)


@pytest.mark.parametrize("k,m", [(256, 256), (129, 70)])
def test_grouped_bad_tables(k, m):
    """Groups outside the output are skipped and sources outside x give zeros, both reported; nothing else changes."""
    w, ws, x, xs = operands(5, 40, k, m, 4)
    out = torch.full((40, m), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = torch.tensor([4, -1, 9, 2], dtype=torch.int32, device="cuda")
    o = torch.tensor([0, 8, 35, -3], dtype=torch.int32, device="cuda")
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, out=out, status=status)
    check_product(out[:4], *product64(w[0], ws[0], x[:4], xs[:4]), k)
    assert torch.all(out[4:] == 5.0) and int(status) == 2
    for big in ([2 ** 31 - 1, 0, 0, 0], [0, 0, 0, 41]):
        status.zero_()
        c = torch.tensor(big, dtype=torch.int32, device="cuda")
        o = torch.tensor([1, 0, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        before = out.clone()
        ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, out=out, status=status)
        assert torch.equal(out, before) and int(status) == 2
    status.zero_()
    rows = torch.arange(40, dtype=torch.int32, device="cuda")
    rows[1], rows[2], rows[3] = -1, 40, 2 ** 31 - 1
    c, o = tables([6, 0, 0, 0])
    out.fill_(5.0)
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, out=out, status=status)
    good = [0, 4, 5]
    check_product(out[good], *product64(w[0], ws[0], x[good], xs[good]), k)
    assert torch.all(out[1:4] == 0) and torch.all(out[6:] == 5.0) and int(status) == 2
    out.fill_(5.0)
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, out=out)  # no status word
    assert torch.all(out[1:4] == 0)
    # the same where the rows are copied first
    many = torch.arange(100, dtype=torch.int32, device="cuda") % 40
    many[1], many[2], many[3] = -1, 40, 2 ** 31 - 1
    c, o = tables([90, 0, 0, 0])
    big = torch.full((100, m), 5.0, device="cuda")
    status.zero_()
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=many, out=big, status=status)
    good = torch.tensor([0] + list(range(4, 90)), device="cuda")
    check_product(big[good], *product64(w[0], ws[0], x[many[good].long()], xs[many[good].long()]), k)
    assert torch.all(big[1:4] == 0) and torch.all(big[90:] == 5.0) and int(status) == 2


def test_grouped_overlapping_tables_end():
    """Groups that lie inside the output one by one but overlap: reported where they add up to more rows than there
    are, never more work than a proper table asks for, nothing outside the output."""
    k, m, e, n = 256, 130, 40, 300
    w, ws, x, xs = operands(2, n, k, m, e)
    c = torch.full((e,), n, dtype=torch.int32, device="cuda")
    o = torch.zeros(e, dtype=torch.int32, device="cuda")
    buf = torch.full((n + 2, m), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, out=buf[1:n + 1], status=status)
    assert int(status) == 2
    assert torch.all(buf[0] == 5.0) and torch.all(buf[n + 1] == 5.0) and torch.isfinite(buf).all()


@pytest.mark.parametrize("k", [256, 253])
def test_grouped_overlap_is_reported_for_any_alignment(k):
    m, e, n = 70, 40, 300
    w, ws, x, xs = operands(3, n, k, m, e)
    c, o = tables([n] + [0] * (e - 1))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, status=status)
    check_product(out, *product64(w[0], ws[0], x, xs), k)
    assert int(status) == 0
    ops.mul_mat_f8_grouped(w, ws, x, xs, torch.full_like(c, n), torch.zeros_like(o), out=out, status=status)
    assert int(status) == 2 and torch.isfinite(out).all()


def test_grouped_fullest_proper_tables_of_any_alignment():
    """As many tiles as groups that do not overlap can have: none of them is refused."""
    for counts in ([1], [64], [65], [1, 1, 1], [65, 65, 65], [64, 1, 64, 1], [63, 66, 128, 129]):
        n, k, m = sum(counts), 37, 66
        w, ws, x, xs = operands(4, n, k, m, len(counts))
        c, o = tables(counts)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, status=status)
        assert int(status) == 0
        for e, (at, cnt) in enumerate(zip(o.tolist(), counts)):
            check_product(out[at:at + cnt], *product64(w[e], ws[e], x[at:at + cnt], xs[at:at + cnt]), k)


# ---------------------------------------------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------------------------------------------
def dequant(q, s, rows=1):
    return q.double() * s.double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]


@pytest.mark.parametrize("n", [1, 6, 70, 300])
def test_feed_forward_layer(n):
    """norm -> gate and up projection -> silu_mul -> down projection, every step against 64 bits on its own inputs."""
    k, f = 512, 768
    g = gen(n)
    x, r = rand(g, n, k).bfloat16(), rand(g, n, k, scale=3.0).bfloat16()
    gamma = (1 + 0.1 * rand(g, k)).bfloat16()
    wgu, sgu = ops.quantize_f8(rand(g, 2 * f, k, scale=0.05), 128)
    wd, sd = ops.quantize_f8(rand(g, k, f, scale=0.05), 128)
    q, s, h = ops.rms_norm_f8(x, gamma, 1e-5, residual=r)
    gu = ops.mul_mat_f8(wgu, sgu, q, s, out_dtype=torch.bfloat16)
    check_product(gu, *product64(wgu, sgu, q, s), k)
    a, sa = ops.silu_mul_f8(gu[:, :f], gu[:, f:])
    y = ops.mul_mat_f8(wd, sd, a, sa, out_dtype=torch.bfloat16)
    check_product(y, *product64(wd, sd, a, sa), f)
    # the whole layer in 64 bits: two roundings to e4m3 and the bf16 ones stay far below the result
    h64 = x.double() + r.double()
    n64 = h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-5) * gamma.double()
    gu64 = n64 @ dequant(wgu, sgu, 128).T
    want = (gu64[:, :f] * torch.sigmoid(gu64[:, :f]) * gu64[:, f:]) @ dequant(wd, sd, 128).T
    assert float((y.double() - want).norm() / want.norm()) < 0.08


@pytest.mark.parametrize("n,e,sel", [(1, 4, 2), (9, 8, 2), (150, 8, 3)])
def test_expert_layer(n, e, sel):
    """moe_route's tables -> gathered up projection -> silu_mul -> down projection on the grouped rows."""
    k, f = 256, 384
    g = gen(n)
    x, sx = ops.quantize_f8(rand(g, n, k))
    wgu, sgu, _, _ = operands(1, 1, k, 2 * f, e)
    wd, sd, _, _ = operands(2, 1, f, k, e)
    ids = torch.rand(n, e, generator=g, device="cuda").topk(sel, 1).indices.to(torch.int32)
    counts, offsets, rows = ops.moe_route(ids, e)
    gu = ops.mul_mat_f8_grouped(wgu, sgu, x, sx, counts, offsets, rows=rows, n_selected=sel)
    a, sa = ops.silu_mul_f8(gu[:, :f], gu[:, f:])
    y = ops.mul_mat_f8_grouped(wd, sd, a, sa, counts, offsets)
    slot = torch.empty_like(y)
    slot[rows.long()] = y
    slot = slot.view(n, sel, k)
    for t in range(n):
        for j in range(sel):
            ei = int(ids[t, j])
            gu64, mags = product64(wgu[ei], sgu[ei], x[t:t + 1], sx[t:t + 1])
            at = int((rows == t * sel + j).nonzero())
            check_product(gu[at:at + 1], gu64, mags, k)
            check_product(slot[t, j][None], *product64(wd[ei], sd[ei], a[at:at + 1], sa[at:at + 1]), f)


def test_other_stream_and_graph():
    """Calls follow the current stream; a captured run gives the bits of an eager one on new inputs."""
    k, m = 1024, 640
    for n in (1, 40, 200):
        g = gen(n)
        w, ws = ops.quantize_f8(rand(g, m, k, scale=0.05), 128)
        x, r, gamma = rand(g, n, k), rand(g, n, k), 1 + 0.1 * rand(g, k)
        counts, offsets = tables([n])
        back = torch.arange(n - 1, -1, -1, dtype=torch.int32, device="cuda")

        def layer():
            q, s, h = ops.rms_norm_f8(x, gamma, 1e-5, residual=r)
            y = ops.mul_mat_f8(w, ws, q, s)
            z = ops.mul_mat_f8_grouped(w[None], ws[None], q, s, counts, offsets)
            z2 = ops.mul_mat_f8_grouped(w[None], ws[None], q, s, counts, offsets, rows=back)
            a, sa = ops.silu_mul_f8(y[:, :m // 2], z[:, m // 2:])
            b, sb = ops.quantize_f8(y)
            return h, y, z, z2, a.float(), sa, b.float(), sb

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = layer()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = layer()
        graph.replay()
        for a, b in zip(first, kept):
            assert torch.equal(a, b)
        x.copy_(rand(g, n, k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(layer(), kept):
            assert torch.equal(a, b)


def test_graph_behind_copies_and_joined_streams():
    """Captured calls whose predecessors are copies, fills and the ends of other streams' work, then each other."""
    g = gen(77)
    n, k, m = 40, 512, 384
    w, ws = ops.quantize_f8(rand(g, m, k, scale=0.05), 128)
    src = [rand(g, n, k) for _ in range(3)]
    x, r, z = (torch.empty(n, k, device="cuda") for _ in range(3))
    gamma = 1 + 0.1 * rand(g, k)
    host = torch.empty(n, m).pin_memory()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()

    def layer():
        here = torch.cuda.current_stream()
        x.copy_(src[0])
        q0, s0 = ops.quantize_f8(x)  # behind a copy
        z.zero_()
        qz, sz = ops.quantize_f8(z)  # behind a fill
        other.wait_stream(here)
        with torch.cuda.stream(other):
            r.copy_(src[1])
            y1 = ops.mul_mat_f8(w, ws, q0, s0)
        y0 = ops.mul_mat_f8(w, ws, qz, sz)
        here.wait_stream(other)
        q, s, h = ops.rms_norm_f8(x, gamma, 1e-5, residual=r)  # behind both streams
        y = ops.mul_mat_f8(w, ws, q, s)
        y1.add_(y)
        host.copy_(y1, non_blocking=True)
        qy, sy = ops.quantize_f8(y1)  # behind a copy to the host
        return y0, y1, h, qy.float(), sy

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = [t.clone() for t in layer()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = layer()
    for _ in range(3):
        for t in (x, r, z, *got):
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(host, want[1].cpu())


def far(t, pitch):
    """A copy of the matrix (or planes) t, the first dimension `pitch` bytes apart."""
    es = t.element_size()
    buf = torch.empty((t.shape[0] - 1) * pitch + t[0].numel() * es, dtype=torch.uint8, device="cuda")
    v = buf.view(t.dtype).as_strided(t.shape, (pitch // es, *t[0].stride()))
    v.copy_(t)
    return v


def test_offsets_past_32_bits():
    """Rows, scales and experts whose byte offsets pass 2^32: the same bits as operands of the same alignment in one
    place give."""
    g, k, m = gen(5), 512, 200
    far3, far20 = (2 << 30) + 4096, (1 << 28) + 4096  # of 3 rows the last, of 20 rows the last four

    x, r = rand(g, 3, k).bfloat16(), rand(g, 3, k).bfloat16()
    gamma = 1 + 0.1 * rand(g, k)
    for pitch in (far3, far3 + 2):  # the second is aligned to elements only
        fx, fr, h = far(x, pitch), far(r, pitch), far(r, pitch)
        near = far(x, 4096 + pitch - far3)  # (a row's sum of squares has an order per alignment)
        out = [far(torch.zeros(3, k, dtype=F8, device="cuda"), pitch), far(torch.zeros(3, k // 128, device="cuda"), far3)]
        for want, got in ((ops.quantize_f8(x), lambda: ops.quantize_f8(fx, out=out[0], scale=out[1])),
                          (ops.silu_mul_f8(x, r), lambda: ops.silu_mul_f8(fx, fr, out=out[0], scale=out[1])),
                          (ops.rms_norm_f8(near, gamma, 1e-5, residual=r)[:2],
                           lambda: ops.rms_norm_f8(fx, gamma, 1e-5, residual=fr, residual_out=h, out=out[0], scale=out[1])[:2])):
            for a, b in zip(got(), want):
                assert torch.equal(a.float(), b.float())
        assert torch.equal(h, x + r)
        del fx, fr, h, out

    w, ws, x, xs = operands(6, 20, k, m)
    for n, pitch in ((3, far3), (20, far20), (20, far20 + 4)):  # GEMV, TMA tiles, any alignment
        fx, fxs, big = far(x[:n], pitch), far(xs[:n], pitch), far(torch.zeros(n, m, device="cuda"), pitch)
        want = ops.mul_mat_f8(far(w, 528 if pitch % 16 == 0 else 516), ws, x[:n], xs[:n])
        got = ops.mul_mat_f8(far(w, 528 if pitch % 16 == 0 else 516), ws, fx, fxs, out=big)
        assert torch.equal(got, want)
        del fx, fxs, big, got
    fw = far(w, 25 << 20)  # 200 rows
    for n in (3, 20):
        assert torch.equal(ops.mul_mat_f8(fw, ws, x[:n], xs[:n]), ops.mul_mat_f8(w, ws, x[:n], xs[:n]))
    del fw

    w, ws, x, xs = operands(7, 24, k, m, 3)
    c, o = tables([4, 0, 20])
    assert torch.equal(ops.mul_mat_f8_grouped(far(w, far3), far(ws, far3), x, xs, c, o),
                       ops.mul_mat_f8_grouped(w, ws, x, xs, c, o))


def test_two_streams_at_once():
    """Products on two streams at the same time share nothing."""
    sets = [operands(s, 30, 4096, 1024) for s in (1, 2)]
    want = [ops.mul_mat_f8(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.mul_mat_f8(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_refusals_on_the_gpu():
    w, ws, x, xs = operands(1, 4, 256, 130)
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    f = torch.zeros(4, 256, device="cuda")
    bad = [
        lambda: ops.mul_mat_f8(w, ws[:1], x, xs), lambda: ops.mul_mat_f8(w, ws, x[:, :128], xs),
        lambda: ops.mul_mat_f8(w, ws, x, xs.double()), lambda: ops.mul_mat_f8(w, ws, f, xs),
        lambda: ops.mul_mat_f8(w, ws, x, xs, out=torch.empty(4, 131, device="cuda")),
        lambda: ops.mul_mat_f8(w, ws, x, xs, out=torch.empty(4, 130, dtype=torch.float64, device="cuda")),
        lambda: ops.mul_mat_f8(w, ws, x, xs.cpu()), lambda: ops.mul_mat_f8(w, ws, x[:1].expand(4, 256), xs),
        lambda: ops.mul_mat_f8(w.view(torch.uint8).t().contiguous().view(F8).t(), ws, x, xs),
        lambda: ops.mul_mat_f8(w, ws, x, xs, out_dtype=torch.int32),
        lambda: ops.mul_mat_f8_grouped(w[None], ws[None], x, xs, i.long(), i),
        lambda: ops.mul_mat_f8_grouped(w[None], ws[None], x, xs, i, i, n_selected=2),
        lambda: ops.mul_mat_f8_grouped(w[None], ws[None], x, xs, i, i, rows=[0]),
        lambda: ops.mul_mat_f8_grouped(w[None], ws[None], x, xs, i, i, rows=i, n_selected=0),
        lambda: ops.quantize_f8(f.double()), lambda: ops.quantize_f8(f[0]), lambda: ops.quantize_f8(f, 64),
        lambda: ops.quantize_f8(f.t()), lambda: ops.quantize_f8(f, out=torch.empty(4, 255, dtype=F8, device="cuda")),
        lambda: ops.rms_norm_f8(f, f[0].bfloat16(), 1e-5), lambda: ops.rms_norm_f8(f, f[0, :5], 1e-5),
        lambda: ops.rms_norm_f8(f, f[0], 1e-5, residual_out=f), lambda: ops.rms_norm_f8(f, f[0], -1.0),
        lambda: ops.rms_norm_f8(f, f[0], 1e-5, residual=f.half()), lambda: ops.silu_mul_f8(f, f.half()),
        lambda: ops.silu_mul_f8(f, f[:3]), lambda: ops.silu_mul_f8(f.view(2, 2, 256), f),
    ]
    for fn in bad:
        with pytest.raises(F.FemlError):
            fn()


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_workspace_refusals(gather):
    """A workspace is checked like every operand, whether the call would use it or not."""
    w, ws, x, xs = operands(1, 40, 256, 130, 1)
    c, o = tables([40])
    rows = torch.arange(40, dtype=torch.int32, device="cuda") if gather else None
    for bad in (b"bytes", torch.empty(20000, dtype=torch.uint8), torch.empty(5000, dtype=torch.int32, device="cuda"),
                torch.empty(100, 200, dtype=torch.uint8, device="cuda"), torch.empty(40000, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(F.FemlError):
            ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, workspace=bad)
