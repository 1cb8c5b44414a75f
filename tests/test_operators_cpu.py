"""CPU: the operators on grouped rows and the gated scan refuse bad arguments before anything is launched, through Python and
through the C ABI; their plans and workspaces are sound over the whole range of sizes; the 64-bit forms that the GPU tests
compare against agree with torch's own autograd."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from test_asan_host import asan_env  # noqa: F401
from util import ROOT
from oracle import operators_oracle as R

LIB = os.environ.get("NERF_TEST_LIB") or os.path.join(ROOT, "nerf_amd", "lib", "libnerf_hip.so")
P = 0x10000          # an address that is only looked at, never read
OK, NULL, SHAPE, ALIGN, WORK, DTYPE = 0, -1, -2, -3, -5, -6


@pytest.fixture(scope="module")
def lib():
    from nerf_amd import _C
    lib = ctypes.CDLL(LIB)
    for name, (res, args) in _C._SIGS.items():
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


def test_cabi_refuses_bad_grouping_arguments(lib):
    f = lib.nerf_group_rows
    need = lib.nerf_group_rows_workspace_bytes(100000, 1000)
    assert lib.nerf_group_rows_workspace_bytes(-1, 5) == lib.nerf_group_rows_workspace_bytes(5, 0) == SHAPE
    assert lib.nerf_group_rows_workspace_bytes(2 ** 31 - 1, 5) == lib.nerf_group_rows_workspace_bytes(5, 2 ** 24 + 1) == SHAPE
    good = [100000, P, 8, 1000, P, P, None, P, need, None]

    def call(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return f(*a)
    assert call(a0=-1) == SHAPE and call(a3=0) == SHAPE and call(a3=2 ** 25) == SHAPE and call(a0=2 ** 31) == SHAPE
    assert call(a2=2) == DTYPE and call(a1=None) == NULL and call(a4=None) == NULL and call(a5=None) == NULL and call(a7=None) == NULL
    assert call(a1=P + 4) == ALIGN and call(a7=P + 64) == ALIGN and call(a8=need - 1) == WORK
    assert f(0, None, 8, 3, None, None, None, None, 0, None) == OK
    g = lib.nerf_group_offsets
    assert g(-1, 3, P, P, P, None) == SHAPE and g(5, 0, P, P, P, None) == SHAPE and g(5, 3, None, P, P, None) == NULL
    assert g(5, 3, P, None, P, None) == NULL and g(5, 3, P, P, None, None) == NULL and g(0, 3, None, None, None, None) == OK


def test_cabi_refuses_bad_table_arguments(lib):
    f, b = lib.nerf_embed_fwd, lib.nerf_embed_bwd
    assert f(-1, P, 8, 5, 8, P, 8, 1.0, 0, P, None) == SHAPE and f(4, P, 8, 0, 8, P, 8, 1.0, 0, P, None) == SHAPE
    assert f(4, P, 8, 5, 0, P, 8, 1.0, 0, P, None) == SHAPE and f(4, P, 8, 5, 8, P, 7, 1.0, 0, P, None) == SHAPE
    assert f(4, P, 8, 5, 2 ** 20 + 1, P, 2 ** 21, 1.0, 0, P, None) == SHAPE
    assert f(4, P, 8, 5, 8, P, 8, 1.0, 3, P, None) == DTYPE and f(4, P, 1, 5, 8, P, 8, 1.0, 0, P, None) == DTYPE
    assert f(4, None, 8, 5, 8, P, 8, 1.0, 0, P, None) == f(4, P, 8, 5, 8, None, 8, 1.0, 0, P, None) == f(4, P, 8, 5, 8, P, 8, 1.0, 0, None, None) == NULL
    assert f(4, P, 8, 5, 8, P + 1, 8, 1.0, 0, P, None) == ALIGN and f(4, P, 8, 5, 8, P + 2, 8, 1.0, 2, P, None) == ALIGN
    assert f(0, None, 8, 5, 8, None, 8, 1.0, 0, None, None) == OK
    need = lib.nerf_embed_bwd_workspace_bytes(5000, 9, 40)
    assert need >= 256 and lib.nerf_embed_bwd_workspace_bytes(-1, 9, 40) == SHAPE and lib.nerf_embed_bwd_workspace_bytes(4096, 1024, 40) == 0
    good = [5000, P, 8, 9, 40, P, 40, 1.0, 0, P, P, need, None]
    for at, bad, code in ((0, -1, SHAPE), (3, 0, SHAPE), (4, 0, SHAPE), (6, 39, SHAPE), (8, 9, DTYPE), (2, 3, DTYPE), (1, None, NULL), (5, None, NULL),
                          (9, None, NULL), (10, None, NULL), (1, P + 4, ALIGN), (5, P + 1, ALIGN), (10, P + 16, ALIGN), (11, need - 1, WORK)):
        a = list(good)
        a[at] = bad
        assert b(*a) == code, at


def test_cabi_refuses_bad_grouped_layer_arguments(lib):
    f, d, w = lib.nerf_grouped_fwd, lib.nerf_grouped_bwd_data, lib.nerf_grouped_bwd_weights
    need = lib.nerf_grouped_bwd_weights_workspace_bytes(5000, 3, 40, 24, 0)
    none = (None, 0, None)                                                     # no workspace, stream
    for G, K, N in ((0, 40, 24), (65536, 40, 24), (3, 0, 24), (3, 40, 0), (3, 65537, 24), (3, 40, 65537)):
        assert f(5000, G, P, P, P, K, N, P, 70000, P, P, 0, 0, P, *none) == SHAPE
        assert d(5000, G, P, P, P, K, N, P, 70000, P, 0, P, *none) == SHAPE
        assert lib.nerf_grouped_bwd_weights_workspace_bytes(5000, G, K, N, 0) == SHAPE == lib.nerf_grouped_workspace_bytes(5000, G, K, N, 0, 0)
        assert w(5000, G, P, P, P, K, N, P, 70000, P, 70000, 0, P, P, P, need, None) == SHAPE
    assert lib.nerf_grouped_bwd_weights_workspace_bytes(5000, 3, 40, 24, 3) == DTYPE == lib.nerf_grouped_workspace_bytes(5000, 3, 40, 24, 1, -1)
    assert f(5000, 3, P, P, P, 40, 24, P, 39, P, P, 0, 0, P, *none) == SHAPE and d(5000, 3, P, P, P, 40, 24, P, 23, P, 0, P, *none) == SHAPE
    assert f(5000, 3, P, P, P, 40, 24, P, 40, P, P, 0, 3, P, *none) == DTYPE and d(5000, 3, P, P, P, 40, 24, P, 24, P, -1, P, *none) == DTYPE
    assert f(5000, 3, None, P, P, 40, 24, P, 40, P, P, 0, 0, P, *none) == NULL
    assert f(5000, 3, P, None, P, 40, 24, P, 40, P, P, 0, 0, P, *none) == NULL and f(5000, 3, P, P, None, 40, 24, P, 40, P, P, 0, 0, P, *none) == NULL
    assert f(5000, 3, P, P, P, 40, 24, P + 1, 40, P, P, 0, 0, P, *none) == ALIGN and d(5000, 3, P, P, P, 40, 24, P, 24, P + 2, 2, P, *none) == ALIGN
    assert w(5000, 3, P, P, P, 40, 24, P, 24, P, 40, 0, P, P, P, need - 1, None) == WORK
    assert w(5000, 3, P, P, P, 40, 24, P, 24, P, 40, 0, P, P, P + 8, need, None) == ALIGN
    assert w(5000, 3, P, P, P, 40, 24, P, 24, P, 40, 0, None, P, P, need, None) == NULL
    assert f(0, 3, None, None, None, 40, 24, None, 40, None, None, 0, 0, None, *none) == OK
    # large products of rows that are not whole pieces need room for copies of them, small ones and whole rows none
    room = lib.nerf_grouped_workspace_bytes
    assert room(500, 3, 41, 24, 1, 2) == room(10 ** 6, 3, 256, 256, 0, 2) == room(10 ** 6, 3, 256, 256, 1, 0) == 0
    fwd, bwd = room(10 ** 6, 3, 67, 250, 0, 2), room(10 ** 6, 3, 67, 250, 1, 2)
    assert 4 * 10 ** 6 * 68 <= fwd <= 4 * (10 ** 6 + 3 * 250) * 68 + 1024 and 4 * 10 ** 6 * 252 <= bwd <= 4 * (10 ** 6 * 252 + 3 * 250 * 68) + 1024
    assert f(10 ** 6, 3, P, P, P, 67, 250, P, 67, P, P, 0, 2, P, P, fwd - 1, None) == WORK
    assert d(10 ** 6, 3, P, P, P, 67, 250, P, 250, P, 2, P, P, bwd - 1, None) == WORK
    assert f(10 ** 6, 3, P, P, P, 67, 250, P, 67, P, P, 0, 2, P, None, fwd, None) == NULL
    assert d(10 ** 6, 3, P, P, P, 67, 250, P, 250, P, 2, P, P + 64, bwd, None) == ALIGN
    r = lib.nerf_relu_bwd
    assert r(-1, 24, P, 24, P, 0, P, None) == r(50, 0, P, 24, P, 0, P, None) == r(50, 24, P, 23, P, 0, P, None) == SHAPE
    assert r(50, 24, P, 24, P, 3, P, None) == DTYPE and r(50, 24, P, 24, P + 1, 0, P, None) == r(50, 24, P, 24, P, 2, P + 2, None) == ALIGN
    assert r(50, 24, None, 24, P, 0, P, None) == r(50, 24, P, 24, None, 0, P, None) == NULL and r(0, 24, None, 24, None, 0, None, None) == OK


def test_cabi_refuses_bad_scan_arguments(lib):
    f, b = lib.nerf_scan_fwd, lib.nerf_scan_bwd
    need = lib.nerf_scan_workspace_bytes(2, 5000, 32, 1, 0, 0)
    good = [2, 5000, 32, P, 5000, 1, 1, P, 160000, 32, None, 0, 0, P, P, None, P, need, None]

    def call(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return f(*a)
    assert call(a0=-1) == call(a1=-1) == call(a2=0) == call(a2=65537) == call(a4=-1) == call(a9=-8) == SHAPE
    assert call(a12=3) == DTYPE and call(a3=None) == call(a7=None) == call(a13=None) == call(a14=None) == call(a16=None) == NULL
    assert call(a7=P + 1) == call(a13=P + 1) == call(a3=P + 1) == call(a14=P + 2) == call(a16=P + 4) == ALIGN and call(a17=need - 1) == WORK
    assert call(a7=P + 2, a8=36001, a9=33, a3=P + 2, a17=0) == WORK            # no more than the elements' own alignment is asked for
    assert f(0, 5, 8, None, 0, 0, 1, None, 0, 0, None, 0, 0, None, None, None, None, 0, None) == OK
    assert lib.nerf_scan_states_floats(2, 5000, 32, 7) == DTYPE and lib.nerf_scan_workspace_bytes(2, 5000, 0, 1, 0, 0) == SHAPE
    need = lib.nerf_scan_workspace_bytes(2, 5000, 32, 1, 1, 0)
    good_b = [2, 5000, 32, P, 5000, 1, 1, P, 160000, 32, None, P, P, P, 0, 0, P, P, P, P, need, None]
    for at, bad, code in ((0, -1, SHAPE), (15, 5, DTYPE), (11, None, NULL), (3, None, NULL), (12, P + 1, ALIGN), (17, P + 1, ALIGN), (20, need - 1, WORK)):
        a = list(good_b)
        a[at] = bad
        assert b(*a) == code, at


def test_plans_are_sound_over_the_range_of_sizes(lib):
    """sizes stay positive, grow at most in proportion and never overflow"""
    for n in (0, 1, 4096, 4097, 10 ** 6, 2 ** 31 - 129):
        for g in (1, 255, 256, 65535, 65536, 2 ** 24):
            assert 256 <= lib.nerf_group_rows_workspace_bytes(n, g) <= 20 * n + 2 ** 16 + 2048 * 4 * (n // 1024 + 3)
            for dim in (1, 7, 64, 1024, 2 ** 20):
                assert (256 if n > 4096 or g > 4096 else 0) <= lib.nerf_embed_bwd_workspace_bytes(n, g, dim) <= 2048 + 28 * n + 4 * g + 2 ** 20 + 8 * 1024 * (n // 1024 + 2) + 8 * dim * (n // 8 + 1)
            if g <= 65535:
                for K, N in ((1, 1), (63, 256), (256, 256), (1024, 1024), (4, 2000), (65536, 65536)):
                    chunks = max(512, (n // 128 + g + 1) // 256 + 1)
                    for prec in (0, 1, 2):
                        b = lib.nerf_grouped_bwd_weights_workspace_bytes(n, g, K, N, prec)
                        a = max(lib.nerf_grouped_workspace_bytes(n, g, K, N, way, prec) for way in (0, 1))
                        assert 256 <= b <= 2048 + 8 * chunks * (N * K + N) + 4 * n * (N + K + 14)
                        assert 0 <= a <= 1024 + 4 * (n + g * N) * (max(K, N) + 7)
    for B in (1, 2, 1000, 10 ** 6):
        for T in (0, 1, 2, 63, 64, 1000, 10 ** 6):
            for D in (1, 3, 64, 67, 256, 4096):
                for prec in (0, 1, 2):
                    s = lib.nerf_scan_states_floats(B, T, D, prec)
                    if T > 2 ** 46 // (B * D):
                        assert s == SHAPE
                        continue
                    assert 0 <= s <= B * T * D
                    for shared in (0, 1):
                        w = lib.nerf_scan_workspace_bytes(B, T, D, shared, 1, prec)
                        assert 256 <= w <= 4 * (3 * B * T * D + (D + 63) // 64 * B * T) + 2048
    assert lib.nerf_scan_states_floats(2 ** 31, 2 ** 40, 64, 0) == SHAPE and lib.nerf_scan_states_floats(2 ** 31, 2 ** 14, 65536, 0) == SHAPE


def test_argument_checks_and_plans_under_sanitizers(asan_env):  # noqa: F811
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", os.path.abspath(__file__), "-k", "cabi or plans_are", "-p", "no:cacheprovider"],
                       env=asan_env, capture_output=True, text=True, timeout=600, cwd=ROOT)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, r.stderr[-3000:]


def test_cpu_tensors_are_refused():
    from nerf_amd import ops
    i, f = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    for call in (lambda: ops.group_rows(i, 2), lambda: ops.row_groups(i, 2), lambda: ops.embed_rows(i, f), lambda: ops.gated_scan(f[None], f[None]),
                 lambda: ops.grouped_linear(f, torch.zeros(2, 3, 8), ops.RowGroups(i, i, i, 4, 2))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: ops.group_rows([0, 1], 2), lambda: ops.embed_rows([0], f), lambda: ops.grouped_linear(f, f, None), lambda: ops.gated_scan(1.0, 2.0)):
        with pytest.raises(TypeError):
            call()


def test_the_64_bit_forms_agree_with_autograd():
    g = torch.Generator().manual_seed(0)
    ids = torch.tensor([2, 0, 2, 9, -1, 1, 2])
    table = torch.randn(4, 3, generator=g, dtype=torch.float64, requires_grad=True)
    d = torch.randn(7, 3, generator=g, dtype=torch.float64)
    ok = (ids >= 0) & (ids < 4)
    want = torch.where(ok[:, None], table[ids.clamp(0, 3)] * 1.5, torch.zeros(()).double())
    assert torch.allclose(R.embed_rows(ids, table, 1.5)[0], want.detach())
    assert torch.allclose(R.embed_rows_grad(ids, 4, d, 1.5)[0], torch.autograd.grad(want, table, d)[0])
    order, offsets = R.group_rows(ids, 4)
    assert order.tolist() == [1, 5, 0, 2, 6, 3, 4] and offsets.tolist() == [0, 1, 2, 5, 5]
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 5), (4, 3, 5), (4, 3)))
    rows_of = [torch.nonzero(ids == e)[:, 0] for e in range(4)]
    z = torch.einsum("rk,rnk->rn", x, w[ids.clamp(0, 3)]) + b[ids.clamp(0, 3)]
    y = torch.relu(z) * ok[:, None]
    got, _ = R.grouped_linear(x, w, b, rows_of, True)
    assert torch.allclose(got, y.detach())
    for (e, _), t in zip(R.grouped_linear_grads(x, w, rows_of, d, got), torch.autograd.grad(y, (x, w, b), d)):
        assert torch.allclose(e, t)
    for shared in (False, True):
        for reverse in (False, True):
            a = torch.randn(2, 6, 1 if shared else 3, generator=g, dtype=torch.float64, requires_grad=True)
            v, s = (torch.randn(q, generator=g, dtype=torch.float64, requires_grad=True) for q in ((2, 6, 3), (2, 3)))
            h, hs = s, {}
            for t in (range(5, -1, -1) if reverse else range(6)):
                h = a[:, t] * h + v[:, t]
                hs[t] = h
            out = torch.stack([hs[t] for t in range(6)], 1)
            dh, dl = torch.randn(2, 6, 3, generator=g, dtype=torch.float64), torch.randn(2, 3, generator=g, dtype=torch.float64)
            ro, _, rl, _ = R.gated_scan(a, v, s, reverse)
            assert torch.allclose(ro, out.detach()) and torch.allclose(rl, h.detach())
            for (e, _), t in zip(R.gated_scan_grads(a, v, s, reverse, dh, dl), torch.autograd.grad((out, h), (a, v, s), (dh, dl))):
                assert torch.allclose(e, t)
