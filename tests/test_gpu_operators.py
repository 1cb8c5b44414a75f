"""GPU: rows grouped by an id (group_rows, row_groups), rows of a table (embed_rows), linear layers of sub-networks
(grouped_linear) and the gated scan against plain 64-bit forms (oracle/operators_oracle.py), at the sizes where tiles,
workgroups and segments begin and end.

Tolerances, derived before the first run.  u = 2^-24 is the largest relative error of one fp32 rounding, r(T) =
finfo(T).eps / 2 that of rounding to T, and `mag` the value's sum taken over absolute values.  A sum of k terms in fp32 in any
order errs by at most k u mag (plus one rounding per product where products are not exact), so every bound here has the form
c u mag + r(T) (|exact| + c u mag) + the smallest step of T, with c the number of fp32 roundings a term can pass through:
  embed forward 1; gradient: rows summed + 1 (the scale);
  grouped_linear: length of the sum + 1 (bias), twice because a matrix instruction's inner additions may truncate;
  scan: a term passes one product and one sum per sample and at most three per level of composition (< 64 levels in all):
  h and d_value 2 T + 192; d_gate is the product of two such values, + the channels it is summed over."""
import math

import pytest
import torch

from util import ROOT  # noqa: F401  (puts the repository on the path)
from oracle import operators_oracle as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def bound(exact, mag, c, dtype):
    f = torch.finfo(dtype)
    err = c * U * mag
    return err + (0.0 if dtype is torch.float32 else f.eps / 2) * (exact.abs() + err) + f.smallest_normal * f.eps + \
        (U * exact.abs() if dtype is torch.float32 else 0.0)


def close(got, exact, mag, c, what=""):
    got64 = got.detach().cpu().double()
    assert got64.shape == exact.shape, (what, got64.shape, exact.shape)
    over = (got64 - exact).abs() - bound(exact, mag, c, got.dtype)
    assert bool((over <= 0).all()), (what, int((~(over <= 0)).sum()), over.max().item(), (got64 - exact).abs().max().item())


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def make_ids(n, groups, kind, g, dtype=torch.int64):
    if kind == "one":
        ids = torch.full((n,), groups // 2)
    elif kind == "none":
        ids = torch.full((n,), -1)
    elif kind == "runs":
        ids = torch.randint(0, groups, ((n + 36) // 37,), generator=g).repeat_interleave(37)[:n]
    elif kind == "skewed":
        ids = (groups * torch.rand(n, generator=g, dtype=torch.float64) ** 4).long().clamp(max=groups - 1)
    else:
        ids = torch.randint(0, groups, (n,), generator=g)
        ids[torch.rand(n, generator=g) < 0.05] = -3
        ids[torch.rand(n, generator=g) < 0.05] = groups
    return ids.to(dtype)


# ---- grouping ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,groups", [(1, 1), (2, 1), (63, 2), (64, 3), (65, 255), (1000, 256), (1025, 257), (2048, 8), (2048, 5000), (2049, 8),
                                      (2049, 300), (300001, 3000), (1100000, 7), (3000001, 5000), (4096, 8), (4096, 5000), (4097, 8), (4097, 255),
                                      (8192, 256), (12289, 70000), (100003, 64), (300000, 1), (50000, 65535)])
def test_group_rows(n, groups, dtype):
    from nerf_amd import ops
    for kind in ("random", "skewed", "one", "none"):
        ids = make_ids(n, groups, kind, gen(n + groups), dtype)
        if dtype is torch.int64 and kind == "random" and n > 2:
            ids[n // 2] = 2 ** 32                                  # not row 0 of a 32-bit id
            ids[n // 3] = -2 ** 62
        order, offsets = R.group_rows(ids, groups)
        got = ops.group_rows(ids.to(DEV), groups)
        assert got.n_rows == n and got.n_groups == groups and got.order.dtype == got.offsets.dtype == torch.int32
        assert torch.equal(got.offsets.cpu().long(), offsets), (kind, "offsets")
        assert torch.equal(got.order.cpu().long(), order), (kind, "order")
        ends = torch.cat([offsets, torch.tensor([n])])
        tiles = torch.cat([torch.zeros(1, dtype=torch.int64), ((ends[1:] - ends[:-1] + 127) // 128).cumsum(0)])
        assert torch.equal(got.tile_base.cpu().long(), tiles), (kind, "tile_base")


def test_group_rows_of_nothing_and_row_groups():
    from nerf_amd import ops
    got = ops.group_rows(torch.zeros(0, dtype=torch.int64, device=DEV), 5)
    assert got.order.numel() == 0 and got.offsets.tolist() == [0] * 6 and got.tile_base.tolist() == [0] * 7
    # boundaries out of order, out of range, beyond 32 bits
    off = torch.tensor([7, 3, 300, 200, -5, 2 ** 40, 500], device=DEV)
    got = ops.row_groups(off, 600)
    assert got.order.tolist() == list(range(600)) and got.offsets.tolist() == [0, 3, 300, 300, 300, 600, 600]
    assert got.tile_base.tolist() == [0, 1, 4, 4, 4, 7, 7, 7]
    big = torch.arange(0, 3001, dtype=torch.int32, device=DEV) * 5
    got = ops.row_groups(big, 20000)
    assert got.offsets.tolist() == [5 * i for i in range(3001)] and got.tile_base[3000].item() == 3000 and got.tile_base[3001].item() == 3040


# ---- rows of a table -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,dim,kind", [(1, 1, 1, "one"), (1024, 100, 48, "random"), (513, 7, 63, "random"), (5000, 9, 3, "skewed"), (30000, 50, 9, "skewed"), (30000, 1, 131, "one"), (20000, 30000, 67, "random"), (3000, 40, 5, "random"),
                                             (40000, 3, 16, "skewed"), (30000, 1, 40, "one"), (3000, 20000, 8, "random"), (70000, 300, 48, "runs"),
                                             (2000, 50, 1000, "random"), (600, 11, 517, "skewed"), (64, 5, 2, "none"), (200000, 4096, 4, "skewed"), (4096, 1024, 20, "random"), (4096, 1025, 20, "random"), (4097, 10, 24, "skewed"),
                                             (3000, 2, 1, "one")])
def test_embed_rows(n, rows, dim, kind, dtype):
    from nerf_amd import ops
    g = gen(n + dim)
    ids = make_ids(n, rows, kind, g)
    table = torch.randn(rows, dim, generator=g).to(dtype)
    d_out = torch.randn(n, dim, generator=g).to(dtype)
    scale = math.sqrt(dim)
    leaf = table.to(DEV).requires_grad_(True)
    out = ops.embed_rows(ids.to(DEV), leaf, scale)
    exact, mag = R.embed_rows(ids, table, scale)
    close(out, exact, mag, 2, "out")
    (d_table,) = torch.autograd.grad(out, leaf, d_out.to(DEV))
    exact, mag, count = R.embed_rows_grad(ids, rows, d_out, scale)
    close(d_table, exact, mag, (count + 2)[:, None].double(), "d_table")
    again = torch.autograd.grad(ops.embed_rows(ids.to(DEV), leaf, scale), leaf, d_out.to(DEV))[0]
    assert torch.equal(d_table, again)                                    # no order of arrival in it


def test_embed_rows_shapes_strides_and_differences():
    from nerf_amd import ops
    g = gen(3)
    wide = torch.randn(20, 40, generator=g).to(DEV)
    for view in (wide[:, :24], wide[:, 3:24], wide[::2, 4:12], wide.t()[:20, :16]):
        ids = torch.randint(-1, view.shape[0] + 1, (4, 5, 3), generator=g).to(torch.int32)
        leaf = view.detach().requires_grad_(True)
        out = ops.embed_rows(ids.to(DEV), leaf, 0.5)
        exact, mag = R.embed_rows(ids, view, 0.5)
        assert out.shape == (4, 5, 3, view.shape[1])
        close(out.reshape(60, -1), exact, mag, 2)
        grad = torch.autograd.grad(out.sum(), leaf)[0]                   # an expanded gradient, strides of zero
        exact, mag, count = R.embed_rows_grad(ids, view.shape[0], torch.ones(60, view.shape[1]), 0.5)
        close(grad, exact, mag, (count + 2)[:, None].double())
        part = torch.autograd.grad(ops.embed_rows(ids.to(DEV), leaf, 0.5)[:, 2:4, :, 1:], leaf, torch.ones(4, 2, 3, view.shape[1] - 1, device=DEV))[0]
        ones = torch.zeros(4, 5, 3, view.shape[1])
        ones[:, 2:4, :, 1:] = 1
        exact, mag, count = R.embed_rows_grad(ids, view.shape[0], ones, 0.5)
        close(part, exact, mag, (count + 2)[:, None].double())
    none = ops.embed_rows(torch.zeros((0, 3), dtype=torch.int64, device=DEV), wide.requires_grad_(True), 2.0)
    assert none.shape == (0, 3, 40)
    assert torch.equal(torch.autograd.grad(none.sum(), wide)[0], torch.zeros_like(wide))
    # differences: the output is linear in the table, so a central difference is exact up to the rounding of the two sums
    table = torch.randn(6, 5, generator=g).to(DEV).requires_grad_(True)
    ids, c = torch.randint(0, 6, (50,), generator=g).to(DEV), torch.randn(50, 5, generator=g).to(DEV)
    grad = torch.autograd.grad(ops.embed_rows(ids, table, 1.5), table, c)[0]
    for r, k in ((0, 0), (3, 4), (5, 2)):
        step = torch.zeros(6, 5, device=DEV)
        step[r, k] = 0.25
        with torch.no_grad():
            two = [(ops.embed_rows(ids, table + s * step, 1.5).double() * c.double()).sum().item() for s in (1, -1)]
        assert abs((two[0] - two[1]) / 0.5 - grad[r, k].item()) < 50 * 4 * U * 8 * 5 / 0.5


def test_embed_rows_keeps_non_finite_values_in_their_rows():
    from nerf_amd import ops
    for n, rows in ((3, 5), (5000, 40), (3, 5000)):                        # rows that nothing reads have no part in an infinite scale
        leaf = torch.ones(rows, 8, device=DEV, requires_grad=True)
        grad = torch.autograd.grad(ops.embed_rows(torch.full((n,), 2, device=DEV), leaf, float("inf")).sum(), leaf)[0]
        assert torch.isinf(grad[2]).all() and grad[:2].eq(0).all() and grad[3:].eq(0).all()
    table = torch.ones(5, 8, device=DEV)
    table[1], table[3] = float("nan"), float("inf")
    out = ops.embed_rows(torch.tensor([0, 1, 2, 3, 7, -1], device=DEV), table, 2.0)
    assert out[0].eq(2).all() and out[1].isnan().all() and out[3].eq(float("inf")).all() and out[4:].eq(0).all()
    assert ops.embed_rows(torch.tensor([9], device=DEV), table, float("nan")).eq(0).all()
    leaf = table.requires_grad_(True)
    d = torch.ones(6, 8, device=DEV)
    d[4], d[0, 2] = float("nan"), float("inf")                            # the gradient of a row that no id names
    grad = torch.autograd.grad(ops.embed_rows(torch.tensor([0, 1, 2, 3, 7, 1], device=DEV), leaf, 2.0), leaf, d)[0]
    assert grad[0, 2] == float("inf") and grad[1].eq(4).all() and grad[4].eq(0).all() and grad[2].eq(2).all()


# ---- linear layers of sub-networks -----------------------------------------------------------------------------------

def linear_case(n, G, K, N, kind, dtype, bias=True, seed=0):
    g = gen(seed + n + K)
    ids = make_ids(n, G, kind, g)
    x = torch.randn(n, K, generator=g).to(dtype)
    w = (torch.randn(G, N, K, generator=g) / math.sqrt(K)).to(dtype)
    b = torch.randn(G, N, generator=g).to(dtype) if bias else None
    d_y = torch.randn(n, N, generator=g).to(dtype)
    rows_of = [torch.nonzero(ids == e)[:, 0] for e in range(G)]
    return ids, x, w, b, d_y, rows_of


def check_linear(x, w, b, d_y, rows_of, groups, relu, xs, ws, bs):
    """xs, ws, bs: the same values on the GPU, leaves"""
    from nerf_amd import ops
    n, K = x.shape
    N = w.shape[1]
    y = ops.grouped_linear(xs, ws, groups, bias=bs, relu=relu)
    exact, mag = R.grouped_linear(x, w, b, rows_of, relu)
    close(y, exact, mag, 2 * (K + 1), "y")
    leaves = [xs, ws] + ([bs] if bs is not None else [])
    got = torch.autograd.grad(y, leaves, d_y.to(DEV))
    want = R.grouped_linear_grads(x, w, rows_of, d_y, y if relu else None)
    counts = torch.tensor([max(1, r.numel()) for r in rows_of]).double()
    for t, (e, m), c, what in zip(got, want, (2 * N, 2 * counts[:, None, None], 2 * counts[:, None]), ("d_x", "d_weight", "d_bias")):
        close(t, e, m, c, what)
    return y, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,G,K,N,kind,relu", [
    (1, 1, 1, 1, "one", False), (1, 3, 63, 256, "one", True), (130, 4, 64, 64, "random", False), (1024, 8, 63, 256, "random", True),
    (1000, 8, 256, 256, "random", True), (257, 2, 27, 3, "skewed", True), (3000, 5, 90, 128, "skewed", False), (512, 700, 16, 24, "random", False),
    (2000, 16, 130, 200, "runs", True), (300, 3, 129, 65, "random", False), (6000, 3, 48, 40, "skewed", True), (200, 2, 512, 384, "random", False),
    (96, 4, 32, 32, "none", True), (9000, 1, 72, 136, "one", False), (140, 65, 8, 8, "runs", False)])
def test_grouped_linear(n, G, K, N, kind, relu, dtype):
    from nerf_amd import ops
    ids, x, w, b, d_y, rows_of = linear_case(n, G, K, N, kind, dtype)
    groups = ops.group_rows(ids.to(DEV), G)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y, got = check_linear(x, w, b, d_y, rows_of, groups, relu, xs, ws, bs)
    none = torch.ones(n, dtype=torch.bool)
    for r in rows_of:
        none[r] = False
    assert y[none.to(DEV)].eq(0).all() and got[0][none.to(DEV)].eq(0).all()
    y2 = ops.grouped_linear(xs, ws, groups, bias=bs, relu=relu)
    again = torch.autograd.grad(y2, [xs, ws, bs], d_y.to(DEV))
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N,relu", [(256, 256, True), (248, 232, False), (40, 1000, False), (1000, 24, True), (67, 256, True), (256, 67, False), (131, 250, True), (9, 1001, False), (1001, 11, True)])
def test_grouped_linear_many_rows(K, N, relu, dtype):
    """enough tiles for the widest output tiles, several tiles per workgroup, some with a ragged last step or last tile"""
    from nerf_amd import ops
    ids, x, w, b, d_y, rows_of = linear_case(60000, 3, K, N, "random", dtype)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    check_linear(x, w, b, d_y, rows_of, ops.group_rows(ids.to(DEV), 3), relu, xs, ws, bs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grouped_linear_long_groups_span_workgroups(dtype):
    """enough rows that every group of the weight gradient is cut over several workgroups, and one that is not"""
    from nerf_amd import ops
    ids, x, w, b, d_y, rows_of = linear_case(150000, 3, 40, 24, "skewed", dtype)
    ids[:100] = 2
    rows_of = [torch.nonzero(ids == e)[:, 0] for e in range(3)]
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    check_linear(x, w, b, d_y, rows_of, ops.group_rows(ids.to(DEV), 3), False, xs, ws, bs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_grouped_linear_strides_no_bias_and_rows_in_order(dtype):
    from nerf_amd import ops
    ids, x, w, _, d_y, _ = linear_case(700, 4, 48, 56, "random", dtype, bias=False)
    off = torch.tensor([0, 100, 100, 431, 650])
    rows_of = [torch.arange(int(off[e]), int(off[e + 1])) for e in range(4)]
    groups = ops.row_groups(off.to(DEV), 700)
    store = torch.zeros(700, 100, dtype=dtype, device=DEV)
    for lo in (0, 8, 3):                                                  # aligned rows, an aligned column block, an unaligned one
        xs = store[:, lo:lo + 48]
        xs.copy_(x)
        xs = xs.detach().requires_grad_(True)
        ws = w.to(DEV).requires_grad_(True)
        y, _ = check_linear(x, w, None, d_y, rows_of, groups, False, xs, ws, None)
        assert y[650:].eq(0).all()
    # leading axes, a transposed x and a transposed weight
    xs = x.to(DEV).t().contiguous().t().requires_grad_(True)
    ws = w.to(DEV).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    check_linear(x, w, None, d_y, rows_of, groups, False, xs, ws, None)
    y = ops.grouped_linear(x.to(DEV).view(7, 100, 48), w.to(DEV), groups)
    assert y.shape == (7, 100, 56)
    # nothing at all
    none = ops.group_rows(torch.zeros(0, dtype=torch.int32, device=DEV), 4)
    xs, ws = torch.zeros(0, 48, dtype=dtype, device=DEV, requires_grad=True), w.to(DEV).requires_grad_(True)
    y = ops.grouped_linear(xs, ws, none)
    dx, dw = torch.autograd.grad(y.sum(), (xs, ws))
    assert y.shape == (0, 56) and dx.shape == (0, 48) and dw.eq(0).all()


def test_grouped_linear_differences():
    """y is linear in each of x, weight and bias: a central difference of a weighted sum is exact up to its rounding"""
    from nerf_amd import ops
    ids, x, w, b, c, _ = linear_case(150, 3, 20, 12, "random", torch.float32)
    groups = ops.group_rows(ids.to(DEV), 3)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.grouped_linear(leaves[0], leaves[1], groups, bias=leaves[2]), leaves, c.to(DEV))
    _, mag = R.grouped_linear(x, w, b, [torch.nonzero(ids == e)[:, 0] for e in range(3)], False)
    room = 2 * 22 * U * (mag * c.double().abs()).sum().item() / 0.5        # the two sums' own errors over the step
    for which, at in ((0, (0, 3)), (0, (149, 19)), (1, (0, 0, 0)), (1, (2, 11, 19)), (2, (1, 5))):
        vals = []
        for s in (0.25, -0.25):
            moved = [t.detach().clone() for t in leaves]
            moved[which][at] += s
            vals.append((ops.grouped_linear(moved[0], moved[1], groups, bias=moved[2]).double().cpu() * c.double()).sum().item())
        assert abs((vals[0] - vals[1]) / 0.5 - grads[which][at].item()) < room + 1e-4 * abs(grads[which][at].item())


@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_keeps_non_finite_rows_apart(dtype):
    from nerf_amd import ops
    ids, x, w, b, d_y, rows_of = linear_case(400, 3, 70, 40, "random", dtype)
    bad = int(rows_of[1][0])
    x[bad] = float("nan")
    out = torch.nonzero((ids < 0) | (ids >= 3))[0, 0].item()
    x[out], d_y[out] = float("inf"), float("nan")                         # a row of no group
    groups = ops.group_rows(ids.to(DEV), 3)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = ops.grouped_linear(xs, ws, groups, bias=bs, relu=True)
    keep = torch.ones(400, dtype=torch.bool)
    keep[bad] = False
    assert y[bad].isnan().all() and y[keep.to(DEV)].isfinite().all() and y[out].eq(0).all()
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), d_y.to(DEV))
    assert dx.isfinite().all() and dx[out].eq(0).all()
    assert dw[0].isfinite().all() and dw[2].isfinite().all() and dw[1].isnan().any() and db.isfinite().all()


# ---- gated scan ------------------------------------------------------------------------------------------------------

def scan_case(B, T, D, gate_shape, dtype, state, seed=0):
    g = gen(seed + B + 7 * T + D)
    gate = torch.exp(-4 * torch.rand(gate_shape, generator=g) ** 6)
    gate = gate * torch.where(torch.rand(gate_shape, generator=g) < 0.1, -1.0, 1.0)
    gate[torch.rand(gate_shape, generator=g) < 0.02] = 0.0
    value = torch.randn(B, T, D, generator=g)
    st = torch.randn(B, D, generator=g) if state else None
    return (gate.to(dtype), value.to(dtype), st, torch.randn(B, T, D, generator=g).to(dtype), torch.randn(B, D, generator=g))


def check_scan(gate, value, st, d_h, d_last, reverse, ga, va, sa):
    from nerf_amd import ops
    B, T, D = value.shape
    c = 2 * T + 192
    h, last = ops.gated_scan(ga, va, state=sa, reverse=reverse)
    e, m, el, ml = R.gated_scan(gate, value, st, reverse)
    close(h, e, m, c, "h")
    close(last, el, ml, c, "last")
    leaves = [ga, va] + ([sa] if sa is not None else [])
    got = torch.autograd.grad((h, last), leaves, (d_h.to(DEV), d_last.to(DEV)))
    want = R.gated_scan_grads(gate, value, st, reverse, d_h, d_last)
    (eg, mg), rest = want[0], want[1:]
    if tuple(eg.shape) != tuple(gate.shape):                               # an expanded axis: autograd adds up our gradients, in T
        for ax in range(2):
            if gate.shape[ax] == 1 and eg.shape[ax] > 1:
                # each of the n terms was rounded to T and so is their sum: n + 1 roundings of T on the magnitude
                n = eg.shape[ax]
                eg, mg = eg.sum(ax, keepdim=True), mg.sum(ax, keepdim=True)
        over = (got[0].cpu().double() - eg).abs() - (2 * c + D) * U * mg - torch.finfo(gate.dtype).eps * (n + 2) * mg
        assert (over <= 0).all()
    else:
        close(got[0], eg, mg, 2 * c + D, "d_gate")
    for t, (e, m), what in zip(got[1:], rest, ("d_value", "d_state")):
        close(t, e, m, c, what)
    return h, last, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 1, 256), (5, 2, 3), (2, 64, 64), (7, 192, 64), (3, 100, 4), (9, 33, 40), (2, 129, 520), (1, 1000, 16),
                                   (4, 257, 67), (300, 5, 8), (1, 20000, 8), (2, 9000, 3), (1, 3000, 256), (2, 1500, 1), (1, 2500, 130), (50, 300, 9), (2, 5000, 13), (6, 70, 8)])
def test_gated_scan(B, T, D, dtype):
    for k, (shared, reverse, state) in enumerate(((True, False, True), (False, True, False), (True, True, False), (False, False, True))):
        if T * B * D > 300000 and k > 1:
            continue
        gate, value, st, d_h, d_last = scan_case(B, T, D, (B, T, 1 if shared else D), dtype, state)
        ga, va = gate.to(DEV).requires_grad_(True), value.to(DEV).requires_grad_(True)
        sa = st.to(DEV).requires_grad_(True) if state else None
        h, last, got = check_scan(gate, value, st, d_h, d_last, reverse, ga, va, sa)
        h2, last2, got2 = check_scan(gate, value, st, d_h, d_last, reverse, ga, va, sa)
        assert torch.equal(h, h2) and torch.equal(last, last2) and all(torch.equal(p, q) for p, q in zip(got, got2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gated_scan_strides_and_expanded_gates(dtype):
    B, T, D = 3, 50, 32
    for shape in ((1, T, 1), (B, 1, 1), (1, 1, D), (1, T, D)):
        gate, value, st, d_h, d_last = scan_case(B, T, D, shape, dtype, True)
        ga, va, sa = (t.to(DEV).requires_grad_(True) for t in (gate, value, st))
        check_scan(gate, value, st, d_h, d_last, False, ga, va, sa)
    gate, value, st, d_h, d_last = scan_case(B, T, D, (B, T, D), dtype, True)
    for make in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),                       # time first in memory
                 lambda t: torch.cat([t, t], 2)[:, :, D:],                                       # a block of channels
                 lambda t: torch.cat([t[:, :, :1], t], 2)[:, :, 1:],                             # one that is not aligned
                 lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):                      # channels not contiguous
        ga, va = make(gate.to(DEV)).detach().requires_grad_(True), make(value.to(DEV)).detach().requires_grad_(True)
        check_scan(gate, value, st, d_h, d_last, True, ga, va, st.to(DEV).requires_grad_(True))


def test_gated_scan_goes_on_from_a_state():
    """one call over all samples, two calls, and a call per sample: the same states up to their rounding"""
    from nerf_amd import ops
    gate, value, st, _, _ = scan_case(4, 300, 24, (4, 300, 24), torch.float32, True)
    e, m, el, ml = R.gated_scan(gate, value, st, False)
    ga, va, sa = gate.to(DEV), value.to(DEV), st.to(DEV)
    for cuts in ((0, 300), (0, 111, 300), tuple(range(301))):
        s, hs = sa, []
        for a, b in zip(cuts[:-1], cuts[1:]):
            h, s = ops.gated_scan(ga[:, a:b], va[:, a:b], state=s)
            hs.append(h)
        close(torch.cat(hs, 1), e, m, 2 * 300 + 192)
        close(s, el, ml, 2 * 300 + 192)


def test_gated_scan_partial_gradients_and_empty_calls():
    from nerf_amd import ops
    gate, value, st, d_h, d_last = scan_case(3, 40, 16, (3, 40, 16), torch.float32, True)
    for pick in range(1, 8):
        leaves = [t.to(DEV).requires_grad_(bool(pick >> i & 1)) for i, t in enumerate((gate, value, st))]
        for use in ((True, False), (False, True), (True, True)):
            h, last = ops.gated_scan(leaves[0], leaves[1], state=leaves[2])
            outs = [o for o, u in zip((h, last), use) if u]
            gs = [o.to(DEV) for o, u in zip((d_h, d_last), use) if u]
            wanted = [t for t in leaves if t.requires_grad]
            got = torch.autograd.grad(outs, wanted, gs)
            want = R.gated_scan_grads(gate, value, st, False, d_h if use[0] else None, d_last if use[1] else None)
            for t, (e, m) in zip(got, [w for i, w in enumerate(want) if pick >> i & 1]):
                close(t, e, m, 2 * (2 * 40 + 192))
    value = torch.zeros(3, 0, 16, device=DEV, requires_grad=True)
    state = st.to(DEV).requires_grad_(True)
    h, last = ops.gated_scan(torch.zeros(3, 0, 1, device=DEV), value, state=state)
    assert h.shape == (3, 0, 16) and torch.equal(last, state)
    assert torch.autograd.grad(last.sum(), state)[0].eq(1).all()
    h, last = ops.gated_scan(torch.zeros(0, 7, 1, device=DEV), torch.zeros(0, 7, 16, device=DEV))
    assert h.shape == (0, 7, 16) and last.shape == (0, 16)


def test_gated_scan_differences():
    """h is affine in any one gate, in the values and in the state: central differences are exact up to rounding"""
    from nerf_amd import ops
    for shared in (False, True):
        gate, value, st, c, cl = scan_case(2, 40, 6, (2, 40, 1 if shared else 6), torch.float32, True)
        leaves = [t.to(DEV).requires_grad_(True) for t in (gate, value, st)]
        grads = torch.autograd.grad(ops.gated_scan(leaves[0], leaves[1], state=leaves[2]), leaves, (c.to(DEV), cl.to(DEV)))
        _, m, _, ml = R.gated_scan(gate.abs() + 0.25, value, st, False)
        room = (2 * 40 + 192) * U * ((m * c.double().abs()).sum() + (ml * cl.double().abs()).sum()).item() / 0.25
        for which, at in ((0, (0, 0, 0)), (0, (1, 39, 0)), (0, (1, 20, 0)), (1, (0, 0, 5)), (1, (1, 39, 2)), (2, (1, 3))):
            vals = []
            for s in (0.25, -0.25):
                moved = [t.detach().clone() for t in leaves]
                moved[which][at] += s
                h, last = ops.gated_scan(moved[0], moved[1], state=moved[2])
                vals.append(((h.cpu().double() * c.double()).sum() + (last.cpu().double() * cl.double()).sum()).item())
            assert abs((vals[0] - vals[1]) / 0.5 - grads[which][at].item()) < room


def test_gated_scan_keeps_non_finite_values_in_their_sequence_and_behind_their_sample():
    from nerf_amd import ops
    for D in (4, 3, 64):
        gate, value, _, d_h, _ = scan_case(6, 90, D, (6, 90, D), torch.float32, False)
        gate = gate.abs().clamp(0.1, 1.0)
        value[2, 31, 1] = float("nan")
        gate[4, 50, 2 % D] = float("inf")
        h, last = ops.gated_scan(gate.to(DEV), value.to(DEV))
        h = h.cpu()
        assert h[:2].isfinite().all() and h[3].isfinite().all() and h[5].isfinite().all()
        assert h[2, :31].isfinite().all() and h[2, 31:, 1].isnan().all() and h[2, :, 0].isfinite().all()
        assert h[4, :50].isfinite().all() and not h[4, 50:, 2 % D].isfinite().any() and h[4, :, 0].isfinite().all()
    # gates above one whose product leaves the range of fp32 while the state is still zero
    gate, value = torch.full((1, 400, 4), 3.0, device=DEV), torch.zeros(1, 400, 4, device=DEV)
    value[:, 390] = 1.0
    h, last = ops.gated_scan(gate, value)
    assert h[:, :390].eq(0).all() and torch.equal(last, torch.full((1, 4), 3.0 ** 9, device=DEV))


# ---- streams, graphs, all of them together ------------------------------------------------------------------------------

def all_ops(ids, table, x, w, b, gate, state, grads):
    """codes per image -> rows dealt out to sub-networks -> two grouped layers -> features composited along the ray"""
    from nerf_amd import ops
    R_, S, K = x.shape
    codes = ops.embed_rows(ids[0], table, 2.0)                              # [rays, code]
    feat = torch.cat([x, codes[:, None].expand(R_, S, codes.shape[-1])], 2).reshape(R_ * S, -1)
    groups = ops.group_rows(ids[1], w[0].shape[0])
    hid = ops.grouped_linear(feat, w[0], groups, bias=b[0], relu=True)
    out = ops.grouped_linear(hid, w[1], groups, bias=b[1]).view(R_, S, -1)
    return ops.gated_scan(gate, out, state=state, reverse=True)


def together(dtype, seed=0, rays=37, S=20):
    g = gen(seed)
    t = {"ids0": torch.randint(0, 9, (rays,), generator=g), "ids1": torch.randint(-1, 5, (rays * S,), generator=g),
         "table": torch.randn(9, 16, generator=g).to(dtype), "x": torch.randn(rays, S, 47, generator=g).to(dtype),
         "w0": (torch.randn(5, 64, 63, generator=g) / 8).to(dtype), "w1": (torch.randn(5, 24, 64, generator=g) / 8).to(dtype),
         "b0": torch.randn(5, 64, generator=g).to(dtype), "b1": torch.randn(5, 24, generator=g).to(dtype),
         "gate": torch.rand(rays, S, 1, generator=g).to(dtype), "state": torch.randn(rays, 24, generator=g),
         "d_h": torch.randn(rays, S, 24, generator=g).to(dtype)}
    return t


NAMES = ("table", "x", "w0", "w1", "b0", "b1", "gate", "state")


def run_together(t):
    leaves = [t[k] for k in NAMES]
    h, last = all_ops((t["ids0"], t["ids1"]), t["table"], t["x"], (t["w0"], t["w1"]), (t["b0"], t["b1"]), t["gate"], t["state"], None)
    grads = torch.autograd.grad((h, last), leaves, (t["d_h"], torch.ones_like(last)))
    return [h.detach(), last.detach()] + list(grads)


def on_gpu(t):
    out = {k: v.to(DEV) for k, v in t.items()}
    for k in NAMES:
        out[k].requires_grad_(True)
    return out


def test_all_operators_together():
    """against torch autograd in 64 bits on the CPU; fp32 operands, so the only difference is rounding: relative to each
    tensor's largest value 1e-4 covers sums of up to 740 rows x 64 features (740 * 64 * u = 3e-3 worst case, 1e-5 as a random
    walk), a unit whose pre-activation is within rounding of zero is kept out by the seed"""
    t = together(torch.float32)
    got = run_together(on_gpu(t))
    c = {k: (v.double() if v.is_floating_point() else v) for k, v in t.items()}
    for k in NAMES:
        c[k].requires_grad_(True)
    codes = 2.0 * c["table"][c["ids0"]]
    feat = torch.cat([c["x"], codes[:, None].expand(-1, 20, -1)], 2).reshape(-1, 63)
    sel = c["ids1"].clamp_min(0)
    ok = (c["ids1"] >= 0).double()[:, None]
    pre = torch.einsum("rk,rnk->rn", feat, c["w0"][sel]) + c["b0"][sel]
    assert pre.abs().min().item() > 1e-6
    hid = torch.relu(pre) * ok
    out = ((torch.einsum("rk,rnk->rn", hid, c["w1"][sel]) + c["b1"][sel]) * ok).view(37, 20, 24)
    h, hs = c["state"], [None] * 20
    for s in range(19, -1, -1):
        h = c["gate"][:, s] * h + out[:, s]
        hs[s] = h
    want = [torch.stack(hs, 1), h]
    grads = torch.autograd.grad(want, [c[k] for k in NAMES], (c["d_h"], torch.ones_like(h)))
    for name, a, b in zip(("h", "last") + NAMES, got, want + list(grads)):
        b = b.detach()
        assert (a.cpu().double() - b).abs().max().item() < 1e-4 * b.abs().max().item(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_graph_replays_equal_eager(dtype):
    """forward and backward of all operators in one HIP graph, replayed on new inputs with eager work in between, two graphs
    captured and alive at once"""
    cases = [on_gpu(together(dtype, s)) for s in range(4)]
    eager = [run_together(c) for c in cases]
    static = [on_gpu(together(dtype, 8)) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_together(static[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            outs.append(run_together(s))
        graphs.append(gph)
    for i in (0, 1, 2, 3, 1, 0):
        for j in (0, 1):
            with torch.no_grad():
                for k, v in static[j].items():
                    v.copy_(cases[(i + j) % 4][k])
        for gph in graphs:
            gph.replay()
        run_together(cases[2])
        torch.cuda.synchronize()
        for j in (0, 1):
            for a, b in zip(outs[j], eager[(i + j) % 4]):
                assert torch.equal(a, b)


def test_calls_on_two_streams():
    cases = [on_gpu(together(torch.bfloat16, s, rays=200, S=64)) for s in range(2)]
    want = [run_together(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, st in zip(cases, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(run_together(c))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


# ---- offsets that pass 32 bits --------------------------------------------------------------------------------------------

def big(shape, dtype):
    """zeros of more than 2^31 elements; the tests put values into the last rows only"""
    assert math.prod(shape) > 2 ** 31
    return torch.zeros(shape, dtype=dtype, device=DEV)


def test_embed_rows_beyond_32_bits():
    from nerf_amd import ops
    n, dim = 2 ** 21 + 5, 1031
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    ids[-3:] = torch.tensor([2, 1, 2], device=DEV)
    table = torch.randn(3, dim, device=DEV, generator=torch.Generator(DEV).manual_seed(0)).half().requires_grad_(True)
    out = ops.embed_rows(ids, table)
    assert torch.equal(out[-4:].detach(), table.detach()[ids[-4:]])
    d_out = big((n, dim), torch.float16)
    d_out[-3:] = torch.randint(-8, 9, (3, dim), device=DEV).half()
    grad = torch.autograd.grad(out, table, d_out)[0]
    assert grad[0].eq(0).all() and torch.equal(grad[1], d_out[-2]) and torch.equal(grad[2], d_out[-3] + d_out[-1])


@pytest.mark.parametrize("K,N", [(1024, 16), (1031, 15)])
def test_grouped_linear_beyond_32_bits(K, N):
    """small whole numbers: every sum is exact, in any order"""
    from nerf_amd import ops
    n = 2 ** 21 + 5
    ids = torch.zeros(n, dtype=torch.int32, device=DEV)
    ids[-3:] = torch.tensor([1, 2, 1], device=DEV, dtype=torch.int32)
    groups = ops.group_rows(ids, 2)
    x = big((n, K), torch.bfloat16)
    x[-4:] = torch.randint(-1, 2, (4, K), device=DEV).bfloat16()
    x.requires_grad_(True)
    w = torch.randint(-1, 2, (2, N, K), device=DEV).bfloat16().requires_grad_(True)
    w.data[:, :, 40:] = 0                                                   # sums of at most 40 terms, whole in bf16
    y = ops.grouped_linear(x, w, groups)
    d_y = torch.zeros_like(y)
    d_y[-4:] = torch.randint(-1, 2, (4, N), device=DEV).bfloat16()
    dx, dw = torch.autograd.grad(y, (x, w), d_y)
    xs, ws, ds = x.detach()[-4:].double(), w.detach().double(), d_y[-4:].double()
    own = (0, 1, None, 1)
    for i, g in enumerate(own):
        assert torch.equal(y[-4 + i].detach().double(), ws[g] @ xs[i] if g is not None else torch.zeros(N, device=DEV).double())
        assert torch.equal(dx[-4 + i].double(), ws[g].t() @ ds[i] if g is not None else torch.zeros(K, device=DEV).double())
    for g in (0, 1):
        assert torch.equal(dw[g].double(), sum(torch.outer(ds[i], xs[i]) for i in range(4) if own[i] == g))
    assert y.detach()[:-4].eq(0).all() and not dx[:-4].any()


@pytest.mark.parametrize("B,T,D", [(2, 2 ** 22 + 3, 256), (2 ** 21 + 1, 4, 260)])
def test_gated_scan_beyond_32_bits(B, T, D):
    """zero gates and one of 1/2: h is the value, and the sample behind the gate adds half the one before it"""
    from nerf_amd import ops
    value = big((B, T, D), torch.bfloat16)
    tail = torch.randint(-8, 9, (3, D), device=DEV).bfloat16()
    value[-1, -3:] = tail
    gate = torch.zeros(B, T, 1, dtype=torch.bfloat16, device=DEV)
    gate[-1, -1] = 0.5
    value.requires_grad_(True), gate.requires_grad_(True)
    h, last = ops.gated_scan(gate, value)
    assert torch.equal(h[-1, -3:-1], tail[:2]) and torch.equal(h[-1, -1], tail[2] + tail[1] / 2) and torch.equal(last[-1], h[-1, -1].float())
    assert h.detach()[-1, :-3].eq(0).all() and h.detach()[:-1].eq(0).all()
    d_h = big((B, T, D), torch.bfloat16)
    g = torch.randint(-8, 9, (2, D), device=DEV).bfloat16()
    d_h[-1, -2:] = g
    d_gate, d_value = torch.autograd.grad(h, (gate, value), d_h)
    assert torch.equal(d_value[-1, -1], g[1]) and torch.equal(d_value[-1, -2], g[0] + g[1] / 2)
    assert d_value[-1, :-2].eq(0).all() and d_value[:-1].eq(0).all()
    want = (g[1].double() * tail[1].double()).sum()                        # whole numbers: exact until the one rounding
    assert d_gate[-1, -1, 0].double() == want.bfloat16().double()


# ---- refusals ---------------------------------------------------------------------------------------------------------

def test_refusals():
    from nerf_amd import ops
    i = torch.zeros(4, dtype=torch.int64, device=DEV)
    f = torch.zeros(4, 8, device=DEV)
    groups = ops.group_rows(i, 2)
    w = torch.zeros(2, 6, 8, device=DEV)
    st = torch.zeros(4, 8, device=DEV)
    v = torch.zeros(4, 5, 8, device=DEV)
    for err, call in (
            (TypeError, lambda: ops.group_rows(f, 2)), (ValueError, lambda: ops.group_rows(i[None], 2)), (ValueError, lambda: ops.group_rows(i, 0)),
            (ValueError, lambda: ops.group_rows(i, 2 ** 25)), (TypeError, lambda: ops.group_rows(i, 2.5)), (TypeError, lambda: ops.row_groups(i, 4.0)), (TypeError, lambda: ops.row_groups(f[0], 4)), (ValueError, lambda: ops.row_groups(i[:1], 4)),
            (ValueError, lambda: ops.row_groups(i, -1)),
            (TypeError, lambda: ops.embed_rows(f, f)), (TypeError, lambda: ops.embed_rows(i, i)), (TypeError, lambda: ops.embed_rows(i, f.double())),
            (ValueError, lambda: ops.embed_rows(i, f[0])), (ValueError, lambda: ops.embed_rows(i, f[:0])), (ValueError, lambda: ops.embed_rows(i, f[:, :0])),
            (TypeError, lambda: ops.embed_rows(i, f, f[0, 0])), (RuntimeError, lambda: ops.embed_rows(i, f.cpu())),
            (TypeError, lambda: ops.grouped_linear(f, w, i)), (TypeError, lambda: ops.grouped_linear(f, w.half(), groups)),
            (TypeError, lambda: ops.grouped_linear(f.double(), w.double(), groups)), (ValueError, lambda: ops.grouped_linear(f, w[0], groups)),
            (ValueError, lambda: ops.grouped_linear(f, torch.zeros(3, 6, 8, device=DEV), groups)), (ValueError, lambda: ops.grouped_linear(f[:3], w, groups)),
            (ValueError, lambda: ops.grouped_linear(f[:, :7], w, groups)), (ValueError, lambda: ops.grouped_linear(f, w, groups, bias=f)),
            (TypeError, lambda: ops.grouped_linear(f, w, groups, bias=torch.zeros(2, 6, device=DEV).half())),
            (RuntimeError, lambda: ops.grouped_linear(f.cpu(), w, groups)),
            (ValueError, lambda: ops.gated_scan(v, f)), (ValueError, lambda: ops.gated_scan(v[:, :3], v)), (ValueError, lambda: ops.gated_scan(v[:, :, :2], v)),
            (ValueError, lambda: ops.gated_scan(v[0], v)), (TypeError, lambda: ops.gated_scan(v.half(), v)), (TypeError, lambda: ops.gated_scan(v, v, state=st.half())),
            (ValueError, lambda: ops.gated_scan(v, v, state=st[:3])), (RuntimeError, lambda: ops.gated_scan(v, v, state=st.cpu())),
            (TypeError, lambda: ops.gated_scan(v.long(), v.long()))):
        with pytest.raises(err):
            call()


def test_second_derivatives_are_refused():
    from nerf_amd import ops
    v = torch.rand(2, 5, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(ops.gated_scan(v, v)[0].sum(), v, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
