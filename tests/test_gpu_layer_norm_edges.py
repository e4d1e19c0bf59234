"""Layer norm on libdvae_hip at the ends of its range."""
import pytest
import torch

import dvae_amd
from util_learn import ln_exact, ln_exact_grad

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


U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def _xhat_bound(x, xh, inv):
    """|computed xh - xh| where nothing but the first sum sees the size of the mean.  That sum goes through `depth` additions, so
    the first mean is off by e = depth u mean|x|; x minus a number that near is exact (Sterbenz) or rounded once.  From there on
    every sum is over distances of |x - mean| + e, again `depth` roundings each: the mean's correction, the variance, whose terms
    are up to (1 + (e / sigma)^2) of it, and in the backward pass the sum of h."""
    c = x.shape[-1]
    depth = max(16, -(-c // 1024)) + 6 + 16
    xd = x.double()
    e = depth * U * xd.abs().mean(-1, keepdim=True)
    away = ((xd - xd.mean(-1, keepdim=True)).abs().mean(-1, keepdim=True) + e) * inv
    return (depth + 6) * U * (away + xh.abs() * (2 + (e * inv).square()))


def _rows(kind, c, dtype):
    g = torch.Generator().manual_seed(c)
    n = torch.randn(5, c, generator=g)
    if kind == "constant":
        x = torch.tensor([0.1, 1.0 / 3.0, -1234.567, 1e6 + 1.0, 7e-3])[:, None].expand(5, c)
    elif kind == "two values":                                       # neighbours in fp32 (bf16): the mean lies between numbers
        low = torch.tensor([0.1, 1.0 / 3.0, -1234.567, 1e6 + 1.0, 7e-3])[:, None].to(dtype).expand(5, c)
        up = torch.nextafter(low.contiguous(), torch.full((5, c), 1e30, dtype=dtype))
        x = torch.where(n > 0.3, up, low)
    else:                                                            # mean over spread 1e5 and 1e6 (bf16: as far as its steps allow)
        x = torch.tensor([1e5, -1e6, 1e4, 3e6, 1e5])[:, None] + n * torch.tensor([1.0, 1.0, 0.1, 4.0, 0.5])[:, None]
        if dtype == torch.bfloat16:
            x = torch.tensor([100.0, -200.0, 50.0, 300.0, 120.0])[:, None] + n
    dy, w, b = torch.randn(5, c, generator=g), 1 + 0.3 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)
    return x.to(dtype).contiguous().cuda(), dy.to(dtype).cuda(), w.cuda(), b.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["constant", "two values", "far mean"])
@pytest.mark.parametrize("c", [5, 31, 193, 512, 777, 4096, 9000, 20001])
def test_rows_whose_mean_is_large_against_their_spread(c, kind, dtype):
    x, dy, w, b = _rows(kind, c, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = dvae_amd.layer_norm(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in leaves)
    alone = torch.autograd.grad(dvae_amd.layer_norm(x, leaves[1], b), leaves[1], dy)[0]      # without dx
    want, xh, inv = ln_exact(x, w, b, 1e-5)
    dx, dw, db = ln_exact_grad(dy, xh, inv, w)
    off = _xhat_bound(x, xh, inv)
    half = HALF_STEP[dtype]
    held(y.detach(), want, off * w.double().abs() + 4 * U * (xh.abs() * w.double().abs() + b.double().abs()) + half * want.abs() + 1e-38)
    # the variance's share of xh's bound is the root's too
    d = max(16, -(-c // 1024)) + 6 + 16
    g = dy.double().abs() * w.double().abs()
    m1, m2, me = (t.mean(-1, keepdim=True) for t in (g, g * xh.abs(), g * off))
    e = d * U * x.double().abs().mean(-1, keepdim=True)
    root = (d + 8) * U * (2 + (e * inv).square())
    inner = (d + 4) * U * (g + m1 + 2 * xh.abs() * m2) + off * m2 + (xh.abs() + off) * me
    held(got[0], dx, inv * inner + root * inv * (g + m1 + xh.abs() * m2) + half * dx.abs() + 1e-38)
    tw = (dy.double().abs() * off).sum(0) + 16 * U * (dy.double().abs() * (xh.abs() + off)).sum(0) + 1e-38
    held(got[1], dw, tw)
    held(alone, dw, tw)
    held(got[2], db, 16 * U * dy.double().abs().sum(0) + 1e-38)
