"""The e4m3 products by the kernel that a shape takes: tile width, persistence, bands of row tiles, cluster splits and
the decode kernel's forms. Every test asserts the plan (148 SMs), so that a later launch rule cannot move the last shape
off a kernel unnoticed. Tolerances: test_gpu_f8.py."""
import math

import pytest
import torch

from feml_b200 import ops
from tests.test_gpu_f8 import F8, TYPES, check_grouped, check_product, gen, operands, product64, tables

pytestmark = pytest.mark.gpu


def plan(k, m, n, experts=0):
    tile, warps, ctas, split = ops.mul_mat_f8_plan(k, m, n, experts)
    return tile, warps, split


# ---------------------------------------------------------------------------------------------------------------
# 256-column tiles
# ---------------------------------------------------------------------------------------------------------------
# one tile per SM and fewer; several tiles per SM; a partial last band of row tiles; K that ends inside a block and
# a chunk of scales; last weight tiles of less and of more than 128 rows; last row tiles of 60, 92, 52 and 68 rows
WIDE = [(700, 272, 3210), (1500, 144, 6500), (2100, 144, 2500), (2500, 1296, 4200), (2500, 1296, 4300)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m", WIDE)
def test_wide_tiles(t, n, k, m):
    assert plan(k, m, n) == (256, 12, 1)
    w, ws, x, xs = operands(n + m, n, k, m)
    got = ops.mul_mat_f8(w, ws, x, xs, out_dtype=t)
    check_product(got, *product64(w, ws, x, xs), k)
    assert torch.equal(got, ops.mul_mat_f8(w, ws, x, xs, out_dtype=t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad,lead", [(1, 0), (3, 1), (8, 0)])
def test_wide_tiles_into_a_wider_buffer(t, pad, lead):
    """Output rows of any alignment; what lies beside them is kept."""
    n, k, m = 700, 272, 3210
    w, ws, x, xs = operands(pad, n, k, m)
    out = torch.full((n + 2, m + pad + lead), 3.0, dtype=t, device="cuda")
    got = ops.mul_mat_f8(w, ws, x, xs, out=out[1:n + 1, lead:lead + m])
    check_product(got, *product64(w, ws, x, xs), k)
    assert torch.all(out[0] == 3.0) and torch.all(out[n + 1] == 3.0)
    assert torch.all(out[:, :lead] == 3.0) and torch.all(out[:, lead + m:] == 3.0)


def test_wide_tiles_strided_scales_and_nan():
    """Scales inside wider matrices; a NaN reaches its own row, its own column or its own block row."""
    n, k, m = 2100, 1296, 2500
    assert plan(k, m, n) == (256, 12, 1)
    w, ws, x, xs = operands(3, n, k, m)
    xs2 = torch.nn.functional.pad(xs, (2, 3), value=math.nan)[:, 2:2 + xs.shape[1]]
    ws2 = torch.nn.functional.pad(ws, (1, 5), value=math.nan)[:, 1:1 + ws.shape[1]]
    got = ops.mul_mat_f8(w, ws2, x, xs2)
    check_product(got, *product64(w, ws, x, xs), k)
    xb, wb, wsn = x.view(torch.uint8).clone(), w.view(torch.uint8).clone(), ws.clone()
    xb[1500, 1295] = 0x7F
    wb[2400, 640] = 0xFF
    wsn[3, 10] = math.nan  # weight rows 384..511
    bad = torch.isnan(ops.mul_mat_f8(wb.view(F8), wsn, xb.view(F8), xs))
    want = torch.zeros_like(bad)
    want[1500] = True
    want[:, 2400] = True
    want[:, 384:512] = True
    assert torch.equal(bad, want)


WIDE_GROUPS = [([1000, 0, 129, 2600, 271], 1296, 1100), ([0, 0, 3000, 0], 1296, 2500)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("counts,k,m", WIDE_GROUPS)
@pytest.mark.parametrize("gather", [False, True])
def test_wide_tiles_grouped(t, counts, k, m, gather):
    """Without a row table, and with one whose rows are copied first."""
    total, gap, e = sum(counts), 5, len(counts)
    n_rows = total + gap + 7
    assert plan(k, m, n_rows, e) == (256, 12, 1)
    c, o = tables(counts, gap)
    n = 300 if gather else n_rows
    w, ws, x, xs = operands(e, n, k, m, e)
    rows = torch.randint(0, 2 * n, (n_rows,), generator=gen(m), device="cuda", dtype=torch.int32) if gather else None
    source = (rows // 2).long() if gather else torch.arange(n_rows, device="cuda")
    out = torch.full((n_rows, m), 5.0, dtype=t, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, n_selected=2 if gather else 1, out=out, status=status)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), source, k)
    assert torch.all(got[:gap] == 5.0) and torch.all(got[gap + total:] == 5.0) and int(status) == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gather", [False, True])
def test_wide_tiles_few_rows_per_expert(t, gather):
    """With a row table the tile's rows are gathered one by one; a bad entry gives zeros."""
    e, n_rows, k, m = 40, 600, 400, 2000
    assert plan(k, m, n_rows, e) == (256, 12, 1) and ops.mul_mat_f8_grouped_workspace(k, n_rows, e) == 0
    counts = torch.randint(0, 25, (e,), generator=gen(2), device="cuda").tolist()
    counts[5], counts[6] = 0, 140
    over = max(0, sum(counts) - n_rows + 4)
    counts[6] -= over
    c, o = tables(counts)
    n = 77 if gather else n_rows
    w, ws, x, xs = operands(11, n, k, m, e)
    rows = torch.randint(0, n, (n_rows,), generator=gen(3), device="cuda", dtype=torch.int32) if gather else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((n_rows, m), 5.0, dtype=t, device="cuda")
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, out=out, status=status)
    total = sum(counts)
    check_grouped(out, w, ws, x, xs, counts, o.tolist(), rows.long() if gather else torch.arange(n_rows, device="cuda"), k)
    assert torch.all(out[total:] == 5.0) and int(status) == 0
    if gather:
        at = int(o[6]) + 130  # a row of the group's second row tile
        rows[at] = n
        want = out.clone()
        want[at] = 0
        ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, out=out, status=status)
        assert torch.equal(out, want) and int(status) == 2


# ---------------------------------------------------------------------------------------------------------------
# clusters that share a tile
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,k,m,split", [(129, 3216, 2500, 2), (100, 3216, 6000, 2), (300, 2064, 1500, 4), (140, 2064, 1500, 4),
                                         (200, 2064, 1000, 8), (17, 2064, 5, 8), (128, 8208, 256, 8)])
def test_split_tiles(t, n, k, m, split):
    assert plan(k, m, n) == (128, 12, split)
    w, ws, x, xs = operands(n + k, n, k, m)
    out = torch.full((n, m + 3), 3.0, dtype=t, device="cuda")  # rows of any alignment
    got = ops.mul_mat_f8(w, ws, x, xs, out=out[:, :m])
    check_product(got, *product64(w, ws, x, xs), k)
    assert torch.all(out[:, m:] == 3.0)
    assert torch.equal(got, ops.mul_mat_f8(w, ws, x, xs, out_dtype=t))


# (experts, counts, k, m, split)
SPLIT_GROUPS = [([70, 0, 100, 0, 0, 31], 3216, 700, 2), ([200, 129, 0], 2064, 500, 4), ([20, 7, 1], 4112, 300, 8), ([0, 20], 4096, 200, 8),
                ([0, 0, 3], 2064, 70, 8)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("counts,k,m,split", SPLIT_GROUPS)
@pytest.mark.parametrize("gather", ["no", "tiles", "copied"])
def test_split_tiles_grouped(t, counts, k, m, split, gather):
    """Groups of clusters: empty groups and clusters past the last group, rows that are kept, rows gathered in the
    product (an empty workspace) or copied before it."""
    e, total, gap = len(counts), sum(counts), 2
    n_rows = total + gap + 4
    assert plan(k, m, n_rows, e) == (128, 12, split)
    c, o = tables(counts, gap)
    n = n_rows if gather == "no" else 41
    w, ws, x, xs = operands(total, n, k, m, e)
    rows = None if gather == "no" else torch.randint(0, 3 * n, (n_rows,), generator=gen(total), device="cuda", dtype=torch.int32)
    source = torch.arange(n_rows, device="cuda") if rows is None else (rows // 3).long()
    work = torch.empty(0, dtype=torch.uint8, device="cuda") if gather == "tiles" else None
    out = torch.full((n_rows, m), 5.0, dtype=t, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, n_selected=1 if rows is None else 3, out=out, workspace=work, status=status)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), source, k)
    assert torch.all(got[:gap] == 5.0) and torch.all(got[gap + total:] == 5.0) and int(status) == 0


@pytest.mark.parametrize("copied", [False, True])
@pytest.mark.parametrize("k,m,split", [(2064, 700, 4), (4112, 130, 8), (3216, 900, 2)])
def test_split_tiles_bad_tables(k, m, split, copied):
    """Groups outside the output are skipped, sources outside x give zeros, both are reported."""
    e = 8 if split == 2 else 4
    n_rows = 200 if copied else 16 * e
    assert plan(k, m, n_rows, e) == (128, 12, split)
    w, ws, x, xs = operands(5, 60, k, m, e)
    rows = torch.arange(n_rows, dtype=torch.int32, device="cuda") % 60
    rows[1], rows[2], rows[9] = -1, 60, 2 ** 31 - 1
    rows[n_rows - 1] = -5  # in no group
    counts = [12, 20, -1, n_rows] + [0] * (e - 4)
    offsets = [0, 30, 4, 1] + [0] * (e - 4)
    c, o = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (counts, offsets))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((n_rows, m), 5.0, device="cuda")
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, o, rows=rows, out=out, status=status)
    assert (ops.mul_mat_f8_grouped_workspace(k, n_rows, e) > 0) == copied
    good = torch.tensor([0, 3, 4, 5, 6, 7, 8, 10, 11], device="cuda")
    check_product(out[good], *product64(w[0], ws[0], x[rows[good].long()], xs[rows[good].long()]), k)
    check_product(out[30:50], *product64(w[1], ws[1], x[rows[30:50].long()], xs[rows[30:50].long()]), k)
    assert torch.all(out[[1, 2, 9]] == 0) and torch.all(out[12:30] == 5.0) and torch.all(out[50:] == 5.0)
    assert int(status) == 2


def test_split_tiles_overlapping_tables_end():
    k, m, e, n = 2064, 130, 5, 130
    assert plan(k, m, n, e)[2] > 1
    w, ws, x, xs = operands(2, n, k, m, e)
    buf = torch.full((n + 2, m), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = torch.full((e,), n, dtype=torch.int32, device="cuda")
    ops.mul_mat_f8_grouped(w, ws, x, xs, c, torch.zeros_like(c), out=buf[1:n + 1], status=status)
    assert int(status) == 2
    assert torch.all(buf[0] == 5.0) and torch.all(buf[n + 1] == 5.0) and torch.isfinite(buf).all()


# ---------------------------------------------------------------------------------------------------------------
# the decode kernel
# ---------------------------------------------------------------------------------------------------------------
# k % 32 == 0: 32-byte loads; else 16-byte ones. n <= 8: one group of rows of x, else two
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [1, 3, 8, 9, 12, 16])
@pytest.mark.parametrize("k,m,warps,split", [(2080, 2500, 16, 1), (2064, 2500, 16, 1), (4128, 9440, 16, 1), (272, 9500, 8, 1),
                                             (288, 9500, 8, 1), (4128, 100, 8, 2), (8208, 64, 8, 4), (8224, 70, 8, 4), (16400, 64, 8, 8),
                                             (16416, 33, 8, 8), (16416, 2000, 8, 2)])
def test_decode(t, n, k, m, warps, split):
    assert plan(k, m, n) == (32, warps, split)
    w, ws, x, xs = operands(n + k + m, n, k, m)
    out = torch.full((n, m + 1), 3.0, dtype=t, device="cuda")
    got = ops.mul_mat_f8(w, ws, x, xs, out=out[:, :m])
    check_product(got, *product64(w, ws, x, xs), k)
    assert torch.all(out[:, m:] == 3.0)


@pytest.mark.parametrize("n", [1, 12])
@pytest.mark.parametrize("k,m", [(2080, 2500), (16400, 64)])
def test_decode_nan(n, k, m):
    """A NaN value or scale reaches its own row, column or block row in every form of the kernel."""
    w, ws, x, xs = operands(n, n, k, m)
    xb, wb, xsn = x.view(torch.uint8).clone(), w.view(torch.uint8).clone(), xs.clone()
    wb[50, k - 1] = 0x7F
    want = torch.zeros(n, m, dtype=torch.bool, device="cuda")
    want[:, 50] = True
    if n > 1:
        xb[3, 77] = 0xFF
        xsn[10, 16] = math.nan
        want[3] = want[10] = True
    assert torch.equal(torch.isnan(ops.mul_mat_f8(wb.view(F8), ws, xb.view(F8), xsn)), want)


# ---------------------------------------------------------------------------------------------------------------
# rows shorter than a block, in whole 16-byte units
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("k", [16, 48, 112])
@pytest.mark.parametrize("n", [1, 16, 17, 140])
def test_short_rows(n, k):
    w, ws, x, xs = operands(n + k, n, k, 200)
    check_product(ops.mul_mat_f8(w, ws, x, xs), *product64(w, ws, x, xs), k)
    c, o = tables([n])
    check_product(ops.mul_mat_f8_grouped(w[None], ws[None], x, xs, c, o), *product64(w, ws, x, xs), k)


def ends(q, fill):
    """q [.., r, k] with rows 16-byte aligned and `fill` behind each row's end."""
    k = q.shape[-1]
    wide = torch.full((*q.shape[:-1], (k + 15) // 16 * 16 + 16), fill, dtype=torch.uint8, device="cuda")
    wide[..., :k] = q.view(torch.uint8)
    return wide.view(F8)[..., :k]


@pytest.mark.parametrize("k", [5, 131, 1299, 2051])
@pytest.mark.parametrize("n,m", [(1, 2500), (12, 200), (40, 200), (300, 300), (700, 3210)])
def test_row_ends_inside_a_vector(n, m, k):
    """Aligned rows whose length is no multiple of 16: the NaN bytes behind their ends count for nothing."""
    w, ws, x, xs = operands(n + k, n, k, m)
    got = ops.mul_mat_f8(ends(w, 0x7F), ws, ends(x, 0xFF), xs)
    check_product(got, *product64(w, ws, x, xs), k)


@pytest.mark.parametrize("k", [5, 1299, 2051])
@pytest.mark.parametrize("work", ["none", "empty", "given"])
def test_row_ends_inside_a_vector_grouped(k, work):
    e, counts, m = 3, [50, 0, 71], 300
    c, o = tables(counts)
    w, ws, x, xs = operands(k, 40, k, m, e)
    rows = torch.randint(0, 40, (121,), generator=gen(k), device="cuda", dtype=torch.int32)
    need = ops.mul_mat_f8_grouped_workspace(k, 121, e)
    room = {"none": None, "empty": torch.empty(0, dtype=torch.uint8, device="cuda"),
            "given": torch.full((need,), 0x7F, dtype=torch.uint8, device="cuda")}[work]
    got = ops.mul_mat_f8_grouped(ends(w, 0x7F), ws, ends(x, 0xFF), xs, c, o, rows=rows, workspace=room)
    check_grouped(got, w, ws, x, xs, counts, o.tolist(), rows.long(), k)


def test_captured_calls_of_every_kernel():
    """One graph with a wide, a split, a gathered and a decode product behind each other: the bits of eager calls."""
    k, m = 2064, 2500
    w, ws, x, xs = operands(1, 2100, k, m)
    rows = torch.arange(60, dtype=torch.int32, device="cuda").flip(0).contiguous()
    c, o = tables([0, 40, 20])
    we, wse = torch.stack([w[:130]] * 3), torch.stack([ws[:2]] * 3)

    def calls():
        a = ops.mul_mat_f8(w, ws, x, xs, out_dtype=torch.bfloat16)
        b = ops.mul_mat_f8(w[:1000], ws[:8], x[:200], xs[:200])
        d = ops.mul_mat_f8_grouped(we, wse, x, xs, c, o, rows=rows)
        e = ops.mul_mat_f8(w, ws, x[:3], xs[:3])
        q, s = ops.quantize_f8(a[:, :k])
        return a, b, d, e, ops.mul_mat_f8(w, ws, q, s)

    assert plan(k, m, 2100)[0] == 256 and plan(k, 1000, 200)[2] == 8 and plan(k, 130, 60, 3)[2] > 1 and plan(k, m, 3)[1] == 16
    want = calls()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(2):
        for t in got:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
