"""GPU: sampling and sorting of more rays than one launch holds (a wave per ray: 2^26 rays are 2^32 threads, and the runtime cuts
off what a direction of a grid has beyond that).  The rays at the beginning, around 2^24 and 2^26 and at the end are compared bit
for bit with the same rays in a small call."""
import pytest
import torch

from util import ROOT  # noqa: F401  (puts the repository on the path)

pytestmark = pytest.mark.gpu
N = 2 ** 26 + 9
DEV = "cuda"


def parts():
    for at in (0, 2 ** 24 - 5, 2 ** 25 + 3, 2 ** 26 - 6, N - 11):
        yield slice(at, at + 11)


def rays(cols, seed):
    return torch.rand(N, cols, device=DEV, generator=torch.Generator(DEV).manual_seed(seed))


def ascending(seed):
    return rays(4, seed).add_(torch.arange(4.0, device=DEV))


def test_sort_rows_of_very_many_rows():
    from nerf_amd import ops
    a, b = rays(2, 0), rays(1, 1)
    out = ops.sort_rows(a, b)
    x, y, z = a[:, 0], a[:, 1], b[:, 0]
    least, most = torch.minimum(torch.minimum(x, y), z), torch.maximum(torch.maximum(x, y), z)
    middle = torch.maximum(torch.minimum(x, y), torch.minimum(torch.maximum(x, y), z))
    assert torch.equal(out[:, 0], least) and torch.equal(out[:, 1], middle) and torch.equal(out[:, 2], most)


@pytest.mark.parametrize("det", [True, False])
def test_sample_pdf_of_very_many_rays(det):
    from nerf_amd import ops
    bins, weights, u = ascending(0), rays(3, 1), None if det else rays(3, 2)
    out, inds = ops.sample_pdf(bins, weights, 3, det=det, u=u, return_inds=True)
    assert out.ge(bins[:, :1] - 1e-5).all() and out.le(bins[:, -1:] + 1e-5).all() and inds.ge(0).all() and inds.le(4).all()
    for s in parts():
        want, winds = ops.sample_pdf(bins[s], weights[s], 3, det=det, u=None if det else u[s], return_inds=True)
        assert torch.equal(out[s], want) and torch.equal(inds[s], winds), s


@pytest.mark.parametrize("det", [True, False])
def test_sample_merge_of_very_many_rays(det):
    from nerf_amd import ops
    z, w, u = ascending(0), rays(4, 1), None if det else rays(2, 2)
    out, fine = ops.sample_merge(z, w, 2, det, u=u, return_fine=True)
    assert out[:, 1:].ge(out[:, :-1]).all() and out[:, 0].eq(torch.minimum(z[:, 0], fine.min(1).values)).all()
    for s in parts():
        want, wfine = ops.sample_merge(z[s], w[s], 2, det, u=None if det else u[s], return_fine=True)
        assert torch.equal(out[s], want) and torch.equal(fine[s], wfine), s
