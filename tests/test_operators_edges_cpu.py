"""CPU: argument checks and plans of the operators' further entry points and forms, beside tests/test_operators_cpu.py."""
import os
import subprocess
import sys

from test_asan_host import asan_env  # noqa: F401
from test_operators_cpu import ALIGN, DTYPE, NULL, OK, P, SHAPE, WORK, lib  # noqa: F401
from util import ROOT


# ---- gates that repeat over sequences or samples ---------------------------------------------------------------------

def test_cabi_refuses_bad_arguments_of_a_repeated_gate(lib):  # noqa: F811
    f, room = lib.nerf_scan_bwd_repeat, lib.nerf_scan_repeat_workspace_bytes
    need, plain = room(2, 5000, 32, 1, 1, 0, 0), lib.nerf_scan_workspace_bytes(2, 5000, 32, 1, 1, 0)
    assert room(2, 5000, 0, 1, 1, 0, 0) == room(-1, 5, 8, 1, 0, 1, 0) == SHAPE and room(2, 5, 8, 1, 1, 1, 3) == DTYPE
    assert room(2, 5000, 32, 1, 0, 0, 0) == plain < need
    good = [2, 5000, 32, P, 0, 1, 1, P, 160000, 32, None, P, P, P, 0, 1, 0, 0, P, P, P, P, need, None]
    for at, bad, code in ((0, -1, SHAPE), (2, 65537, SHAPE), (5, -1, SHAPE), (17, 5, DTYPE), (11, None, NULL), (3, None, NULL), (7, None, NULL),
                          (21, None, NULL), (12, P + 1, ALIGN), (18, P + 1, ALIGN), (21, P + 4, ALIGN), (22, need - 1, WORK)):
        a = list(good)
        a[at] = bad
        assert f(*a) == code, at
    a = list(good)
    a[18], a[22] = None, plain - 1                                          # no gradient of the gate: no room for its terms either
    assert f(*a) == WORK
    assert f(0, 5, 8, None, 0, 0, 1, None, 0, 0, None, None, None, None, 0, 1, 1, 0, None, None, None, None, 0, None) == OK


def test_plans_of_repeated_gates_are_sound(lib):  # noqa: F811
    """room for the fp32 terms and at most as much again for sums of runs of eight terms or more"""
    for B in (1, 2, 1000, 10 ** 6, 2 ** 31):
        for T in (1, 2, 63, 1000, 10 ** 6):
            for D in (1, 3, 64, 67, 4096):
                for prec in (0, 1, 2):
                    for shared in (0, 1):
                        base = lib.nerf_scan_workspace_bytes(B, T, D, shared, 1, prec)
                        for over_b, over_t in ((1, 0), (0, 1), (1, 1)):
                            w = lib.nerf_scan_repeat_workspace_bytes(B, T, D, shared, over_b, over_t, prec)
                            if base < 0:
                                assert w == SHAPE
                                continue
                            terms = B * T * (1 if shared else D)
                            assert base + 4 * terms <= w <= base + 8 * terms + 1024 + 4 * 2048 * 256


def test_checks_and_plans_under_sanitizers(asan_env):  # noqa: F811
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", os.path.abspath(__file__), "-k", "cabi or plans_of", "-p", "no:cacheprovider"],
                       env=asan_env, capture_output=True, text=True, timeout=600, cwd=ROOT)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, r.stderr[-3000:]
