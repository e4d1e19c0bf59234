"""Newton-Schulz and the Muon step at sizes that take each of the batched kernels: symmetric products straight from memory, in tiles
of 64 and 128, whole and in pieces, and the last product in tiles of 64, of 128 and of 128 shared by two groups of waves.
The 64-bit iteration runs on the device."""
import math

import pytest
import torch

import dvae_amd
from util_learn import COEF, HALF_STEP, ns

pytestmark = pytest.mark.gpu


def gradient(m, n, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g)
    x += 4.0 / math.sqrt(max(m, n)) * torch.randn(m, 3, generator=g) @ torch.randn(3, n, generator=g)
    return (1e-3 * x).to(dtype).cuda()


def bound(x):
    """64-bit result and the tolerance of a part of it: eight times the float32 iteration's error there, 2^-20 of the part and the
    rounding to x's type."""
    want, yard = ns(x.double()), ns(x.float()).double()
    half = HALF_STEP[x.dtype] if x.dtype != torch.float32 else 0.0
    return want, lambda d, part: 8 * float((yard - want)[part].norm()) + (2.0 ** -20 + half) * float(want[part].norm()) + 1e-30


def held(got, x):
    """In tiles of 64 x 64 and the ragged ones at the edges: a tile that is wrong, missing or in another's place shows."""
    want, tol = bound(x)
    d = got.double() - want
    assert got.shape == want.shape and got.dtype == x.dtype
    m, n = x.shape
    assert float(d.norm()) <= tol(d, slice(None))
    tiles = lambda v: torch.nn.functional.pad(v.square(), (0, -n % 64, 0, -m % 64)).unflatten(1, (-1, 64)).unflatten(0, (-1, 64)).sum((1, 3)).sqrt()   # noqa: E731
    yard = (ns(x.float()).double() - want)
    half = HALF_STEP[x.dtype] if x.dtype != torch.float32 else 0.0
    # of a tile on its own the float32 error is a draw: its mean square over all tiles, and sixteen times it
    typical = float(yard.norm()) / math.sqrt(tiles(yard).numel())
    assert bool((tiles(d) <= 16 * (tiles(yard) + typical) + (2.0 ** -19 + half) * tiles(want)).all())


ONE = [(512, 4608), (2048, 2048), (1984, 2048), (2048, 1984), (1984, 2050), (1024, 4608), (4608, 1000), (1500, 2500), (700, 5000), (130, 20000),
       (200, 60000), (1024, 2048), (2900, 2900), (1030, 1031)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", ONE)
def test_one_matrix(m, n, dtype):
    x = gradient(m, n, m + n, dtype)
    got = dvae_amd.newton_schulz(x)
    held(got, x)
    assert torch.equal(got, dvae_amd.newton_schulz(x))                # the same bits again


@pytest.mark.parametrize("m,n", [(4608, 512), (60000, 200)])
def test_transposes_agree(m, n):
    x = gradient(m, n, 3)
    y = dvae_amd.newton_schulz(x.t().contiguous())
    held(dvae_amd.newton_schulz(x), x)
    assert torch.equal(dvae_amd.newton_schulz(y.t()).t(), dvae_amd.newton_schulz(y))


@pytest.mark.parametrize("shapes", [[(1024, 1024)] * 16, [(512, 4608)] * 4 + [(256, 2304)] * 3 + [(512, 256), (10, 512), (64, 27)],
                                    [(700, 700)] * 9, [(256, 2304)] * 12, [(2048, 2048), (1984, 1990), (100, 90)], [(4096, 4096), (64, 64)]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lists(shapes, dtype):
    xs = [gradient(m, n, i, dtype) for i, (m, n) in enumerate(shapes)]
    out = dvae_amd.newton_schulz(xs)
    for x, y in list(zip(xs, out))[:4] + list(zip(xs, out))[-4:]:
        held(y, x)


def _step_held(p, g, m, lr, decay, mu=0.95):
    want = []
    for pp, gg, mm in zip(p, g, m):
        p64, g64, m64 = pp.double(), gg.double(), mm.double()
        m64 = mu * m64 + (1 - mu) * g64
        u = (1 - mu) * g64 + mu * m64
        if pp.dim() < 2:
            want.append((p64 * (1 - lr * decay) - lr * u, m64, 4 * lr * HALF_STEP[torch.float32] * float(u.norm()) + 3 * 2.0 ** -24 * float(p64.norm())))
            continue
        u = u.reshape(pp.shape[0], -1)
        s = math.sqrt(max(1.0, u.shape[0] / u.shape[1]))
        w = ns(u)
        # u is off by four roundings of fp32, which the iteration amplifies as it does the yardstick's rounded start
        yard = (ns(u.float()).double() - w).norm() + 4 * (ns(u.float().double()) - w).norm()
        want.append((p64 * (1 - lr * decay) - lr * s * w.view(pp.shape), m64,
                     lr * s * (8 * float(yard) + 2.0 ** -19 * float(w.norm())) + 3 * 2.0 ** -24 * float(p64.norm())))
    dvae_amd.muon_step(p, g, m, lr=lr, momentum=mu, weight_decay=decay)
    for (w, m64, tol), pp, mm in zip(want, p, m):
        assert float((pp.double() - w).norm()) <= tol, (tuple(pp.shape), float((pp.double() - w).norm()), tol)
        assert float((mm.double() - m64).norm()) <= 4 * 2.0 ** -24 * float(m64.norm()) + 1e-30


@pytest.mark.parametrize("shapes", [[(512, 512, 3, 3)], [(2048, 2048)], [(1984, 2048)], [(1000, 4000), (77,)], [(512, 512, 3, 3)] * 4 + [(512,), (256, 256, 3, 3), (10, 512)],
                                    [(1024, 1024)] * 16, [(4608, 512)]])
def test_muon_step(shapes):
    """From zero parameters, so that nothing but the step is compared, with a gradient and a momentum of one size."""
    p = [torch.zeros(s, device="cuda") for s in shapes]
    mk = lambda k: [gradient(s[0], math.prod(s[1:]), 7 * i + k).view(s) if len(s) > 1 else 1e-3 * torch.ones(s, device="cuda") for i, s in enumerate(shapes)]   # noqa: E731
    _step_held(p, mk(0), mk(1), lr=0.02, decay=0.01)


def test_classifier_steps_all_its_weights():
    """The 512-row weights of layer4 among the classifier's 62 parameters, from real gradients."""
    torch.manual_seed(0)
    model = dvae_amd.ResNet18(10).cuda().train()
    x, y = torch.rand(8, 3, 32, 32, device="cuda"), torch.arange(8, device="cuda")
    torch.nn.functional.cross_entropy(model(x), y).backward()
    params = [p.detach().clone() for p in model.parameters()]
    _step_held(params, [p.grad.clone() for p in model.parameters()], [torch.zeros_like(p) for p in params], lr=0.02, decay=0.0)
