"""GPU: the operators of nerf_amd.ops at their edges, beside tests/test_gpu_operators.py.

Most operands here are small whole numbers (or halves), so that every sum is exact in fp32 in any order as long as its
magnitude stays below 2^24 steps of its smallest term: results are compared bit for bit with the exact value rounded once,
and a single missing, repeated or misplaced row shows."""
import math

import pytest
import torch

from util import ROOT  # noqa: F401  (puts the repository on the path)
from oracle import operators_oracle as R
from test_gpu_operators import DEV, DTYPES, U, close, gen, scan_case

pytestmark = pytest.mark.gpu


def whole(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g).float()


# ---- forward-mode derivatives ----------------------------------------------------------------------------------------

def test_forward_mode_is_refused_not_dropped():
    """A tensor with a tangent has requires_grad False; a result without a tangent would count as a derivative of zero."""
    import torch.autograd.forward_ad as fw
    from nerf_amd import ops
    ids = torch.tensor([0, 2, 1, 0], device=DEV)
    table = torch.randn(3, 8, device=DEV)
    groups = ops.group_rows(ids, 3)
    x, w, b = torch.randn(4, 8, device=DEV), torch.randn(3, 5, 8, device=DEV), torch.randn(3, 5, device=DEV)
    gate, value, state = torch.rand(2, 6, 8, device=DEV), torch.randn(2, 6, 8, device=DEV), torch.randn(2, 8, device=DEV)
    calls = [(lambda t: ops.embed_rows(ids, t), table),
             (lambda t: ops.grouped_linear(t, w, groups, bias=b, relu=True), x), (lambda t: ops.grouped_linear(x, t, groups, bias=b), w),
             (lambda t: ops.grouped_linear(x, w, groups, bias=t), b), (lambda t: ops.grouped_linear(t, w, groups), x.view(2, 2, 8)),
             (lambda t: ops.gated_scan(t, value), gate), (lambda t: ops.gated_scan(t, value), gate[:1, :, :1]),
             (lambda t: ops.gated_scan(gate, t, state=state), value), (lambda t: ops.gated_scan(gate, value, state=t, reverse=True), state)]
    for mode in (torch.enable_grad, torch.no_grad):
        for call, t in calls:
            with mode(), fw.dual_level(), pytest.raises(NotImplementedError):
                call(fw.make_dual(t, torch.ones_like(t)))
        with mode(), fw.dual_level():                                      # nothing carries a tangent: an ordinary call
            for call, t in calls:
                a, b2 = call(t), call(t)
                assert all(torch.equal(p, q) for p, q in zip(a, b2))
    for call, t in calls:
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
        out = call(t.detach().requires_grad_(True))
        out = out[0] if isinstance(out, tuple) else out
        with fw.dual_level(), pytest.raises(NotImplementedError):          # nor are those of an incoming gradient
            out.backward(fw.make_dual(torch.ones_like(out), torch.ones_like(out)))
        out.backward(torch.ones_like(out))


# ---- gates that repeat over sequences or samples ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [(3, 50, 32), (65, 3, 40), (1, 700, 9), (700, 1, 8), (5, 333, 3), (2, 4000, 130), (300, 40, 1), (2, 30, 1031)])
def test_gated_scan_gradient_of_a_repeated_gate_is_summed_in_fp32(B, T, D, dtype):
    """d_gate is a sum over B and / or T as well: its terms, the fp32 values of the full gate's gradient (2 (2 T + 192) + D
    roundings, tests/test_gpu_operators.py), meet in fp32, at most one rounding per term, and are rounded to the type once"""
    from nerf_amd import ops
    for k, shape in enumerate(((1, T, 1), (B, 1, 1), (1, 1, 1), (1, T, D), (B, 1, D), (1, 1, D))):
        gate, value, st, d_h, d_last = scan_case(B, T, D, shape, dtype, True)
        ga, va, sa = (t.to(DEV).requires_grad_(True) for t in (gate, value, st))
        runs = []
        for _ in range(2):
            h, last = ops.gated_scan(ga, va, state=sa, reverse=bool(k & 1))
            runs.append(torch.autograd.grad((h, last), (ga, va, sa), (d_h.to(DEV), d_last.to(DEV))))
        (eg, mg), (ev, mv), (es, ms) = R.gated_scan_grads(gate, value, st, bool(k & 1), d_h, d_last)
        terms = 1
        for ax in range(2):
            if gate.shape[ax] != eg.shape[ax]:
                terms *= eg.shape[ax]
                eg, mg = eg.sum(ax, keepdim=True), mg.sum(ax, keepdim=True)
        c = 2 * T + 192
        got = runs[0][0]
        assert got.dtype == dtype and got.shape == shape
        # A sum from (2 - eps / 2) 2^e on, 2^e the type's largest power of two, is nearer to the first value behind the type's
        # range than to the last one in it, so its rounding is infinite (fp16: 65 520); within the fp32 sum's error of that
        # border it may be either.
        f = torch.finfo(dtype)
        border, err = (2 - f.eps / 2) * 2.0 ** math.floor(math.log2(f.max)), (2 * c + D + terms) * U * mg
        beyond = got.isinf().cpu() & (eg.abs() + err >= border) & (got.cpu() * eg.sign() > 0)
        assert bool((beyond | (eg.abs() - err < border)).all())
        close(torch.where(beyond.to(DEV), 0, got), torch.where(beyond, 0, eg), torch.where(beyond, 0, mg), 2 * c + D + terms, "d_gate")
        close(runs[0][1], ev, mv, c, "d_value")
        close(runs[0][2], es, ms, c, "d_state")
        assert all(torch.equal(p, q) for p, q in zip(*runs))


@pytest.mark.parametrize("shape", [(1, 1, 16), (1, 64, 16), (64, 1, 16), (1, 1, 1), (1, 64, 1), (64, 1, 1)])
def test_gated_scan_repeated_gate_outside_the_range_of_a_term(shape):
    """Zero gates: d_gate[t] = d_h[t] h[t-1] = d_h[t] value[t-1].  Terms of 2^-26, below fp16, add up to what it holds; terms of
    +-2^17, beyond it, cancel."""
    from nerf_amd import ops
    gate = torch.zeros(shape, dtype=torch.float16, device=DEV, requires_grad=True)
    full = (64, 64, shape[2])
    for size, grad, sign in ((2.0 ** -13, 2.0 ** -13, False), (512.0, 256.0, True)):
        value = torch.full((64, 64, 16), size, dtype=torch.float16, device=DEV)
        d_h = torch.full((64, 64, 16), grad, dtype=torch.float16, device=DEV)
        if sign:
            d_h[1::2, ::2] *= -1
            d_h[::2, 1::2] *= -1                                           # + - + - along both axes, as many of each
            d_h[:, -1] = 0
        terms = d_h.double() * torch.cat([torch.zeros(64, 1, 16, device=DEV).half(), value[:, :-1]], 1).double()
        if shape[2] == 1:
            terms = terms.sum(2, keepdim=True)
        assert terms.shape == full
        for ax in range(2):
            if shape[ax] == 1:
                terms = terms.sum(ax, keepdim=True)
        got = torch.autograd.grad(ops.gated_scan(gate, value)[0], gate, d_h)[0]
        assert torch.equal(got, terms.half())


def test_repeated_gates_in_a_captured_graph():
    """the sum over samples and sequences takes two launches here; replayed on new inputs with eager work in between"""
    from nerf_amd import ops
    def run(t):
        h, last = ops.gated_scan(t[0], t[1], state=t[2])
        return list(torch.autograd.grad((h, last), t[:3], (t[3], t[4])))
    cases = [[t.to(DEV) for t in scan_case(3, 900, 24, (1, 1, 24), torch.bfloat16, True, seed)] for seed in range(3)]
    static = [t.clone() for t in cases[0]]
    for t in (*cases, static):
        for leaf in t[:3]:
            leaf.requires_grad_(True)
    want = [run(t) for t in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for i in (1, 2, 0, 2):
        with torch.no_grad():
            for a, b in zip(static, cases[i]):
                a.copy_(b)
        graph.replay()
        run(cases[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


# ---- what a group table may hold ---------------------------------------------------------------------------------------

def test_row_groups_checks_its_fields_and_keeps_them():
    import copy
    import pickle
    from nerf_amd import ops
    good = ops.group_rows(torch.tensor([1, 0, 7, 1, 1], device=DEV), 2)
    order, offsets, base = good.order, good.offsets, good.tile_base
    for err, args in ((TypeError, (order.long(), offsets, base, 5, 2)), (TypeError, (order, offsets.float(), base, 5, 2)),
                      (TypeError, (order, offsets, [0, 1, 2, 3], 5, 2)), (ValueError, (order[:4], offsets, base, 5, 2)),
                      (ValueError, (order, offsets, base, 6, 2)), (ValueError, (order, offsets, base, 5, 1)), (ValueError, (order, offsets, base[1:], 5, 2)),
                      (ValueError, (order[None], offsets, base, 5, 2)), (ValueError, (order, offsets, base, -1, 2)), (ValueError, (order, offsets, base, 5, 0)),
                      (TypeError, (order, offsets, base, 5.0, 2)), (RuntimeError, (order, offsets.cpu(), base, 5, 2)), (RuntimeError, (order.cpu(), offsets, base, 5, 2))):
        with pytest.raises(err):
            ops.RowGroups(*args)
    for name in ("order", "offsets", "tile_base", "n_rows", "n_groups", "other"):
        with pytest.raises(AttributeError):
            setattr(good, name, order)
        with pytest.raises(AttributeError):
            delattr(good, name)
    x, w = torch.randn(5, 8, device=DEV), torch.randn(2, 3, 8, device=DEV)
    want = ops.grouped_linear(x, w, good)
    wide = torch.stack([order, order], 1)[:, 0]                            # not contiguous
    for other in (ops.RowGroups(wide, offsets, base, 5, 2), copy.copy(good), copy.deepcopy(good), pickle.loads(pickle.dumps(good))):
        assert torch.equal(ops.grouped_linear(x, w, other), want) and (other.n_rows, other.n_groups) == (5, 2)


def bad_tables(n, G, g):
    """tables of the right size that no grouping gives: of other rows, out of order, out of range"""
    from nerf_amd import ops
    most = n // 128 + G + 1
    other = ops.group_rows(torch.randint(0, G, (n,), generator=g).to(DEV) // 2, G)
    good = ops.group_rows(torch.randint(0, G, (n,), generator=g).to(DEV), G)
    i32 = dict(dtype=torch.int32, device=DEV)
    full = lambda size, v: torch.full((size,), v, **i32)
    wild = lambda size: torch.randint(-2 ** 31, 2 ** 31, (size,), generator=g).to(torch.int32).to(DEV)
    yield "boundaries of other rows", good.order, other.offsets, good.tile_base
    yield "tiles of other rows", good.order, good.offsets, other.tile_base
    yield "boundaries backwards", good.order, good.offsets.flip(0), good.tile_base
    yield "tiles backwards", good.order, good.offsets, good.tile_base.flip(0)
    yield "positions behind the rows", good.order, good.offsets + n, good.tile_base
    yield "tiles behind the last", good.order, good.offsets, good.tile_base + most
    yield "twice the tiles", good.order, good.offsets, good.tile_base * 2
    yield "nothing below zero", good.order, full(G + 1, -1), full(G + 2, -1)
    yield "all at the top", good.order, full(G + 1, 2 ** 31 - 1), full(G + 2, 2 ** 31 - 1)
    yield "all at the bottom", good.order, full(G + 1, -2 ** 31), full(G + 2, -2 ** 31)
    yield "rows that are none", wild(n), good.offsets, good.tile_base
    yield "anything", wild(n), wild(G + 1), wild(G + 2)
    yield "tiles in any order", good.order, good.offsets, torch.randint(0, most + 1, (G + 2,), generator=g).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,G,K,N", [(1000, 8, 256, 256), (500, 70, 63, 40), (40000, 3, 64, 128), (40000, 3, 67, 40), (3000, 80, 128, 64), (300, 2, 64, 64)])
def test_grouped_linear_stays_inside_its_tensors_whatever_the_tables_hold(n, G, K, N, dtype):
    """the C entry points on outputs and workspaces that lie between guards; every kernel ends, nothing outside is written.  (What
    the kernels do with such tables is bounded in groups.hpp: checked_tiles, checked_span.)"""
    from nerf_amd import ops
    from nerf_amd._C import check, lib
    g = gen(n + K)
    code, size = ops._ELEM[dtype], torch.finfo(dtype).bits // 8
    x, w, b, d_y = (torch.randn(s, generator=g).to(dtype).to(DEV) for s in ((n, K), (G, N, K), (G, N), (n, N)))
    guard, st = 1 << 16, torch.cuda.current_stream().cuda_stream
    room = lib.nerf_grouped_bwd_weights_workspace_bytes(n, G, K, N, code)
    areas = {name: torch.empty(bytes_ + 2 * guard, dtype=torch.uint8, device=DEV)
             for name, bytes_ in (("y", n * N * size), ("dx", n * K * size), ("dw", G * N * K * size), ("db", G * N * size), ("work", room))}
    at = {name: a.data_ptr() + guard for name, a in areas.items()}
    nf, nb = (lib.nerf_grouped_workspace_bytes(n, G, K, N, way, code) for way in (0, 1))
    small = torch.empty(max(nf, nb, 256), dtype=torch.uint8, device=DEV)
    for what, order, offsets, base in bad_tables(n, G, g):
        print(what, n, G, K, N, dtype, flush=True)
        for a in areas.values():
            a.fill_(0x5a)
        t = ops.RowGroups(order, offsets, base, n, G)
        p = (n, G, t.order.data_ptr(), t.offsets.data_ptr(), t.tile_base.data_ptr(), K, N)
        check(lib.nerf_grouped_fwd(*p, x.data_ptr(), K, w.data_ptr(), b.data_ptr(), 1, code, at["y"], small.data_ptr(), nf, st), "fwd")
        check(lib.nerf_grouped_bwd_data(*p, d_y.data_ptr(), N, w.data_ptr(), code, at["dx"], small.data_ptr(), nb, st), "bwd_data")
        check(lib.nerf_grouped_bwd_weights(*p, d_y.data_ptr(), N, x.data_ptr(), K, code, at["dw"], at["db"], at["work"], room, st), "bwd_weights")
        torch.cuda.synchronize()
        for name, a in areas.items():
            assert a[:guard].eq(0x5a).all() and a[-guard:].eq(0x5a).all(), (what, name)


# ---- tables written into between forward and backward ------------------------------------------------------------------

def test_grouped_linear_refuses_a_backward_of_other_groups():
    """as torch does for any tensor that a backward needs"""
    from nerf_amd import ops
    x, w = torch.randn(300, 16, device=DEV), torch.randn(4, 8, 16, device=DEV)
    ids = torch.randint(-1, 4, (300,), device=DEV)
    for field in ("order", "offsets", "tile_base"):
        for relu in (False, True):
            for leaf in (0, 1):
                groups = ops.group_rows(ids, 4)
                ops_in = [x.clone(), w.clone()]
                ops_in[leaf].requires_grad_(True)
                y = ops.grouped_linear(*ops_in, groups, relu=relu)
                again = ops.grouped_linear(*ops_in, groups, relu=relu)
                (want,) = torch.autograd.grad(y.sum(), ops_in[leaf])       # the same groups for several calls
                y2 = ops.grouped_linear(*ops_in, groups, relu=relu)
                getattr(groups, field).copy_(getattr(ops.group_rows(3 - ids, 4), field))
                for late in (again, y2):
                    with pytest.raises(RuntimeError, match="modified by an inplace"):
                        late.sum().backward()
                getattr(groups, field).copy_(getattr(ops.group_rows(ids, 4), field))
                y3 = ops.grouped_linear(*ops_in, groups, relu=relu)        # written into before the forward: in order
                assert torch.equal(torch.autograd.grad(y3.sum(), ops_in[leaf])[0], want)


def test_groups_made_in_inference_mode_train():
    from nerf_amd import ops
    x, w, b = torch.randn(300, 16, device=DEV), torch.randn(4, 8, 16, device=DEV), torch.randn(4, 8, device=DEV)
    ids = torch.randint(-1, 4, (300,), device=DEV)
    with torch.inference_mode():
        inside = ops.group_rows(ids, 4)
    got = []
    for groups in (inside, ops.group_rows(ids, 4)):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = ops.grouped_linear(leaves[0], leaves[1], groups, bias=leaves[2], relu=True)
        got.append([y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))])
    assert all(torch.equal(p, q) for p, q in zip(*got))


# ---- layers of the largest sizes that the documentation allows -------------------------------------------------------

def test_grouped_linear_gradient_of_the_largest_layer():
    """65 536 x 65 536 features: more than 2^32 sums in d_weight, of a group that has rows and of one that has none"""
    from nerf_amd import ops
    n, F = 130, 65536
    ids = torch.ones(n, dtype=torch.int32, device=DEV)
    ids[3] = -1
    x = torch.randint(-2, 3, (n, F), device=DEV, generator=torch.Generator(DEV).manual_seed(0)).bfloat16()
    w = torch.zeros(2, F, F, dtype=torch.bfloat16, device=DEV)
    w[1, -1, :40] = 1                                                       # one row and one column: sums of few terms
    w[1, :, -1] = 2
    w.requires_grad_(True)
    bias = torch.zeros(2, F, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = ops.grouped_linear(x, w, ops.group_rows(ids, 2), bias=bias)
    keep = torch.arange(n, device=DEV) != 3
    want = (2 * x[:, -1:].float()).repeat(1, F)
    want[:, -1] += x[:, :40].float().sum(1)
    assert torch.equal(y.detach(), torch.where(keep[:, None], want, 0 * want).bfloat16())
    d_y = torch.zeros(n, F, dtype=torch.bfloat16, device=DEV)
    for i, cols in ((0, slice(0, 7)), (3, slice(0, None)), (5, slice(40000, 40100)), (129, slice(F - 3, None)), (64, slice(F - 1, None))):
        d_y[i, cols] = torch.randint(-3, 4, d_y[i, cols].shape, device=DEV).bfloat16()
    torch.cuda.empty_cache()
    dirt = torch.full((2, F, F), 7.0, dtype=torch.bfloat16, device=DEV)     # what the gradient's memory held before
    del dirt
    dw, db = torch.autograd.grad(y, (w, bias), d_y)
    d_y[3] = 0
    assert torch.equal(db[1], d_y.float().sum(0).bfloat16()) and not db[0].any() and not dw[0].any()
    for lo in range(0, F, 4096):
        rows = d_y[:, lo:lo + 4096].float()
        assert torch.equal(dw[1, lo:lo + 4096], (rows.t().contiguous() @ x.float()).bfloat16()), lo


def test_grouped_linear_most_groups_times_most_outputs():
    """65 535 groups of 65 536 outputs: more than 2^24 tiles of output, most of them of groups without rows"""
    from nerf_amd import ops
    n, G, N = 300, 65535, 65536
    ids = torch.randint(0, G, (n,), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    ids[:4] = torch.tensor([G - 1, 0, -1, G - 1], device=DEV)
    w = torch.zeros(G, N, 1, dtype=torch.bfloat16, device=DEV)
    w[ids.clamp_min(0)] = torch.randint(-4, 5, (n, N, 1), device=DEV).bfloat16()
    x = torch.randint(-4, 5, (n, 1), device=DEV).bfloat16()
    x.requires_grad_(True)
    y = ops.grouped_linear(x, w, ops.group_rows(ids, G))
    ok = (ids >= 0)[:, None]
    assert torch.equal(y.detach(), torch.where(ok, x.detach() * w[ids.clamp_min(0), :, 0], torch.zeros((), device=DEV, dtype=torch.bfloat16)))
    d_y = torch.zeros(n, N, dtype=torch.bfloat16, device=DEV)
    d_y[:, -9:] = torch.randint(-2, 3, (n, 9), device=DEV).bfloat16()
    dx = torch.autograd.grad(y, x, d_y)[0]
    assert torch.equal(dx, torch.where(ok, (w[ids.clamp_min(0), -9:, 0].float() * d_y[:, -9:].float()).sum(1, keepdim=True), torch.zeros((), device=DEV)).bfloat16())


# ---- scans of more sequences than one launch holds -------------------------------------------------------------------

@pytest.mark.parametrize("B,D,dtype", [(2 ** 29 + 3, 7, torch.bfloat16), (2 ** 30 + 1, 3, torch.float16)])
def test_gated_scan_of_very_many_sequences(B, D, dtype):
    """a step of more sequences than one launch holds"""
    from nerf_amd import ops
    g = torch.Generator(DEV).manual_seed(2)
    value = torch.randint(-8, 9, (B, 1, D), device=DEV, generator=g, dtype=torch.int8).to(dtype).requires_grad_(True)
    state = torch.randint(-8, 9, (B, D), device=DEV, generator=g, dtype=torch.int8).float()
    gate = torch.randint(-2, 3, (B, 1, 1), device=DEV, generator=g, dtype=torch.int8).to(dtype).requires_grad_(True)
    h, last = ops.gated_scan(gate, value, state=state)
    d_h = torch.randint(-4, 5, (B, 1, D), device=DEV, generator=g, dtype=torch.int8).to(dtype)
    d_gate, d_value = torch.autograd.grad(h, (gate, value), d_h)
    for lo in range(0, B, 2 ** 27):
        s = slice(lo, lo + 2 ** 27)
        want = gate.detach()[s, 0].float() * state[s] + value.detach()[s, 0].float()
        assert torch.equal(h.detach()[s, 0].float(), want) and torch.equal(last[s], want), lo
        assert torch.equal(d_value[s], d_h[s]), lo
        assert torch.equal(d_gate[s, 0], (d_h[s, 0].float() * state[s]).sum(1, keepdim=True).to(dtype)), lo


# ---- weight gradients and products of many rows, exactly ---------------------------------------------------------------

def exact_layer(offsets, n, K, N, dtype, seed=0):
    """every output and gradient of a layer on whole numbers, bit for bit; offsets: the groups, rows in order"""
    from nerf_amd import ops
    g = gen(seed + n + K)
    G = len(offsets) - 1
    x, w, d_y = whole(g, -2, 2, n, K), whole(g, -1, 1, G, N, K), whole(g, -1, 1, n, N)
    b = whole(g, -3, 3, G, N)
    x[torch.rand(n, generator=g) < 0.5] *= -1
    xs, ws, bs = (t.to(dtype).to(DEV).requires_grad_(True) for t in (x, w, b))
    y = ops.grouped_linear(xs, ws, ops.row_groups(torch.tensor(offsets, device=DEV), n), bias=bs)
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), d_y.to(dtype).to(DEV))
    y, dx, dw, db = (t.detach().cpu() for t in (y, dx, dw, db))
    assert 2 * n < 2 ** 24 and 2 * K < 2 ** 24 and N < 2 ** 24             # every partial sum is exact in fp32
    for e in range(G):
        r = slice(offsets[e], offsets[e + 1])
        assert torch.equal(y[r], (x[r] @ w[e].T + b[e]).to(dtype)), (e, "y")
        assert torch.equal(dx[r], (d_y[r] @ w[e]).to(dtype)), (e, "d_x")
        assert torch.equal(dw[e], (d_y[r].T @ x[r]).to(dtype)), (e, "d_weight")
        assert torch.equal(db[e], d_y[r].sum(0).to(dtype)), (e, "d_bias")
    assert y[offsets[-1]:].eq(0).all() and dx[offsets[-1]:].eq(0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,N", [(40, 24), (64, 64), (67, 40), (131, 250), (256, 256), (40, 1000)])
def test_grouped_linear_every_row_counts(K, N, dtype):
    """groups cut over many workgroups, one that lies inside a single one, empty ones and one of a single row"""
    exact_layer([0, 45000, 45000, 45090, 45091, 59000, 59000], 60000, K, N, dtype)


@pytest.mark.parametrize("K,N,dtype", [(512, 1024, torch.bfloat16), (1024, 512, torch.float16), (256, 256, torch.float32), (255, 257, torch.bfloat16)])
def test_grouped_linear_long_runs_of_tiles_per_workgroup(K, N, dtype):
    """more tiles per workgroup than it keeps row numbers of (24 in the weight gradient, 8 or 12 in the products): groups end one
    tile before, at and behind the places where the numbers are read anew, on ragged tiles and whole ones"""
    tiles = [23, 1, 1, 22, 1, 24, 48, 1, 95, 24, 25, 200, 2, 24]
    offsets = [0]
    for i, t in enumerate(tiles):
        offsets.append(offsets[-1] + t * 128 - (0, 5, 127, 64)[i % 4])
    offsets.append(195000)
    exact_layer(offsets, 200003, K, N, dtype)


# ---- as many groups and table rows as there may be -----------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 100, 2048, 2049, 300001])
def test_group_rows_of_the_most_groups(n):
    """ids of 25 bits: four digits in one workgroup, three in blocks"""
    from nerf_amd import ops
    G = 2 ** 24
    ids = torch.randint(-1, G + 1, (n,), generator=gen(n))
    ids[n // 2:] = ids[n // 2:] % 1000 + G - 1000
    key = torch.where((ids >= 0) & (ids < G), ids, G)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(G + 1))
    for dtype in (torch.int32, torch.int64):
        got = ops.group_rows(ids.to(dtype).to(DEV), G)
        assert torch.equal(got.order.cpu().long(), order) and torch.equal(got.offsets.cpu().long(), offsets)
        ends = torch.cat([offsets, torch.tensor([n])])
        tiles = torch.cat([torch.zeros(1, dtype=torch.int64), ((ends[1:] - ends[:-1] + 127) // 128).cumsum(0)])
        assert torch.equal(got.tile_base.cpu().long(), tiles)


@pytest.mark.parametrize("n,dim", [(5000, 3), (300, 9), (100000, 16)])
def test_embed_rows_of_the_longest_table(n, dim):
    from nerf_amd import ops
    rows = 2 ** 24
    g = gen(n)
    ids = torch.randint(0, rows, (n,), generator=g)
    ids[::3] = rows - 1 - ids[::3] % 5
    ids[0], ids[n // 2] = -1, rows
    table = torch.randint(-8, 9, (rows, dim), generator=torch.Generator(DEV).manual_seed(0), device=DEV).bfloat16().requires_grad_(True)
    d_out = whole(g, -1, 1, n, dim).bfloat16().to(DEV)
    ids = ids.to(DEV)
    ok = (ids >= 0) & (ids < rows)
    out = ops.embed_rows(ids, table, 0.5)
    assert torch.equal(out.detach(), torch.where(ok[:, None], 0.5 * table.detach()[ids.clamp(0, rows - 1)], torch.zeros((), device=DEV).bfloat16()))
    grad = torch.autograd.grad(out, table, d_out)[0]
    want = torch.zeros(rows, dim, device=DEV, dtype=torch.float64).index_add_(0, ids[ok], 0.5 * d_out[ok].double())
    assert torch.equal(grad, want.bfloat16())


# ---- long sums of the table's gradient in fp32 -----------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [128, 20, 3])
def test_embed_rows_gradient_of_half_a_million_terms(dim):
    """A term passes at most 64 additions in its lane group, G in LDS (G = 256 threads / lanes of a row), n / (span G) + 1 over
    workgroups of span = 64 G positions or less and G more, and the scale: far fewer than the terms of the sum."""
    from nerf_amd import ops
    n = 524288
    g = gen(dim)
    d_out = torch.randn(n, dim, generator=g) + 0.25                       # a sum that grows, with terms of either sign
    leaf = torch.zeros(3, dim, device=DEV, requires_grad=True)
    ids = torch.ones(n, dtype=torch.int64)
    ids[::1000] = 2
    grad = torch.autograd.grad(ops.embed_rows(ids.to(DEV), leaf, 2.0), leaf, d_out.to(DEV))[0]
    lanes = 4
    while lanes < 64 and lanes * (4 if dim >= 4 else 1) < dim:
        lanes *= 2
    groups = 256 // lanes
    per = min(64, max(8, (n // (groups * 1024) + 7) // 8 * 8))
    most = per + groups + (n // (groups * per) + groups) // groups + 1 + groups + 1
    exact, mag, _ = R.embed_rows_grad(ids, 3, d_out, 2.0)
    err = (grad.cpu().double() - exact).abs()[1:] / mag[1:]
    print(f"dim {dim}: {most} roundings at most, worst error {err.max().item():.2e} of the magnitude, {((grad.cpu().double() - exact).abs() / exact.abs())[1].max().item():.2e} of the value")
    close(grad, exact, mag, most)
    assert grad[0].eq(0).all()


# ---- states carried over long distances, exactly -------------------------------------------------------------------------

def long_scan(B, T, D, shared, dtype, seed=0):
    """Gates of +-1 with a factor of 2 or 1/2 now and then (in turn, so that products stay within 1 and 2) and whole values:
    h[t] = P[t] (state + sum_{s <= t} value[s] / P[s]) with P the running product of the gates, exactly"""
    g = gen(seed + T + D)
    C = 1 if shared else D
    sign = torch.randint(0, 2, (B, T, C), generator=g) * 2 - 1
    step = torch.rand(B, T, C, generator=g) < 20.0 / T
    scale = torch.where(step, torch.where(step.cumsum(1) % 2 == 1, 2.0, 0.5), 1.0)
    gate = (sign * scale).double()
    some = 200.0 / T                                                      # few enough that the sums stay small
    value, state, d_h, d_last = (torch.where(torch.rand(s, generator=g) < max(some, 1.0 if len(s) == 2 else 0.0),
                                             torch.randint(0, 2, s, generator=g) * 2 - 1, 0).double()
                                 for s in ((B, T, D), (B, D), (B, T, D), (B, D)))
    P = gate.cumprod(1)
    assert P.abs().max() <= 2 and P.abs().min() >= 1
    total = state[:, None] + (value / P).cumsum(1)
    h = P * total
    before = torch.cat([state[:, None], h[:, :-1]], 1)
    # G[t] P[t] = sum_{s >= t} d_h[s] P[s] + d_last P[T-1]
    G = ((d_h * P).flip(1).cumsum(1).flip(1) + (d_last * P[:, -1])[:, None]) / P
    d_gate = G * before
    if shared:
        d_gate = d_gate.sum(2, keepdim=True)
    d_state = gate[:, 0] * G[:, 0]
    # terms are whole, halves at the least (quarters in products), and no partial sum reaches 2^24 of them
    assert 4 * (value.abs().sum(1).max() + d_h.abs().sum(1).max() + 2).item() < 2 ** 22
    assert 4 * (G * before).abs().sum(2).max().item() < 2 ** 24
    return gate, value, state, d_h, d_last, h, d_gate, G, d_state


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1000, 16), (1, 20000, 8), (2, 9000, 3), (2, 5000, 13), (1, 40001, 256), (2, 12000, 64), (1, 20000, 64), (1, 2500, 130), (9, 700, 67),
                                   (1, 300000, 1)])
def test_gated_scan_carries_the_state_to_the_far_end(B, T, D, dtype):
    from nerf_amd import ops
    from nerf_amd._C import lib
    code = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]
    tiles = lib.nerf_scan_states_floats(B, T, D, code) // (B * D) + 1
    if (B, T) == (1, 40001):
        assert tiles > 512                                                # two tiles a segment: more than 256 segments
    for shared in (True, False):
        for reverse in (False, True):
            gate, value, state, d_h, d_last, h, d_gate, d_value, d_state = long_scan(B, T, D, shared, dtype)
            along = (lambda t: t.flip(1)) if reverse else (lambda t: t)
            ga, va = (along(t).to(dtype).to(DEV).requires_grad_(True) for t in (gate, value))
            sa = state.float().to(DEV).requires_grad_(True)
            got_h, last = ops.gated_scan(ga, va, state=sa, reverse=reverse)
            grads = torch.autograd.grad((got_h, last), (ga, va, sa), (along(d_h).to(dtype).to(DEV), d_last.float().to(DEV)))
            assert torch.equal(last.detach().cpu().double(), h[:, -1]), "last"
            assert torch.equal(got_h.detach().cpu(), along(h).to(dtype)), "h"
            assert torch.equal(grads[1].cpu(), along(d_value).to(dtype)), "d_value"
            assert torch.equal(grads[2].cpu().double(), d_state), "d_state"
            assert torch.equal(grads[0].cpu(), along(d_gate).to(dtype)), "d_gate"


# ---- where the scan's range ends -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,shared", [(4, True), (3, False), (64, True)])
def test_gated_scan_products_of_gates_up_to_the_range_of_fp32(D, shared):
    """100 gates in a row whose product is 2^+-120: every state is a power of two and exact, forward and backward"""
    from nerf_amd import ops
    for up in (1, -1):
        gate = torch.ones(1, 100, 1 if shared else D, device=DEV)
        gate[:, 10:70] = 2.0 ** (2 * up)                                   # 60 samples
        gate.requires_grad_(True)
        state = torch.full((1, D), 2.0 ** (-60 * up), device=DEV, requires_grad=True)
        h, last = ops.gated_scan(gate, torch.zeros(1, 100, D, device=DEV), state=state)
        want = state.detach()[0, 0].item() * gate.detach()[0, :, 0].double().cumprod(0)
        assert torch.equal(h.detach()[0].double(), want[:, None].expand(100, D)) and last.detach().eq(2.0 ** (60 * up)).all()
        d_state = torch.autograd.grad(last, state, torch.full((1, D), 2.0 ** (-60 * up), device=DEV))[0]
        assert d_state.eq(2.0 ** (60 * up)).all()
