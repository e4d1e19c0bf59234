"""Layer norm on libdvae_hip at the ends of its range."""
import pytest
import torch

import dvae_amd

pytestmark = pytest.mark.gpu


def held(got, want, tol):
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= tol).all()), (float((d / tol).max()), float(d.max()))


@pytest.mark.parametrize("c", [(1 << 27) - 3, (1 << 27) + 70, 1 << 28])
def test_rows_whose_column_sums_exceed_one_launch(c):
    """From 2^27 columns on a workgroup for every 64 sums would be 2^32 threads and more.  One row: the parameters' gradients
    are dy xh and dy, column by column; every column is compared, in pieces that keep the 64-bit values small."""
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(1, c, device="cuda", generator=g, dtype=torch.bfloat16).requires_grad_(True)
    dy = torch.randn(1, c, device="cuda", generator=g, dtype=torch.bfloat16)
    w, b = torch.ones(c, device="cuda", requires_grad=True), torch.zeros(c, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(dvae_amd.layer_norm(x, w, b), (w, b), dy)
    xd = x.detach().double()
    mean, var = xd.mean(), xd.var(unbiased=False)
    inv = (var + 1e-5).rsqrt()
    size = xd.abs().mean()
    del xd
    assert torch.equal(db, dy[0].float())
    for lo in range(0, c, 1 << 25):
        part = slice(lo, min(c, lo + (1 << 25)))
        xp = x.detach()[0, part].double()
        xh = (xp - mean) * inv
        # the mean is off by at most 2^17 + 22 roundings (a thread's chain of additions) of mean|x|, corrected by its distances' sum
        # that is as long; the variance by as many of itself
        chain = (c // 1024 + 22) * 2.0 ** -24
        tol = dy[0, part].double().abs() * (2 * chain * size * inv + (chain + 8 * 2.0 ** -24) * xh.abs()) + 1e-38
        held(dw[part], dy[0, part].double() * xh, tol)
