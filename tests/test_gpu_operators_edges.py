"""GPU: the operators of nerf_amd.ops at their edges, beside tests/test_gpu_operators.py.

Most operands here are small whole numbers (or halves), so that every sum is exact in fp32 in any order as long as its
magnitude stays below 2^24 steps of its smallest term: results are compared bit for bit with the exact value rounded once,
and a single missing, repeated or misplaced row shows."""
import pytest
import torch

from util import ROOT  # noqa: F401  (puts the repository on the path)
from oracle import operators_oracle as R
from test_gpu_operators import DEV, DTYPES, close, gen, scan_case

pytestmark = pytest.mark.gpu


def whole(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g).float()


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
