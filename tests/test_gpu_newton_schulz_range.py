"""Newton-Schulz on libdvae_hip where parts of a matrix, or all of it, are small: held row by row and column by column."""
import pytest
import torch

import dvae_amd
from util_learn import COEF, HALF_STEP, ns

pytestmark = pytest.mark.gpu
A5 = COEF[0]


def noise(m, n, seed):
    return torch.randn(m, n, generator=torch.Generator().manual_seed(seed)).cuda()


def floor_of(m, n, steps):
    """What fp16 pieces leave of absolute errors, as the norm of a row (of p or q): an element of X is off by at most 2^-50 where
    its pieces have no digits left, one of A or B by 2^-49.  A row of X takes q (p) of the former; a row of B its own p, those
    of b A (4.8 times) and of c A^2 (twice, times |A| <= 4, times 2.03), times |X| <= 2.  A step's errors grow by a^(steps left)."""
    p, q = min(m, n), max(m, n)
    return 2.0 ** -49 * (q ** 0.5 / 2 + 44 * p ** 0.5) * A5 ** steps / (A5 - 1)


def held_everywhere(x, steps=5, eps=1e-7):
    """Every row and every column within eight times the worst relative one of the same iteration in float32 (22 bits against 24 and
    sums as long), 2^-19 of itself, the rounding to its type, and the absolute floor."""
    got = dvae_amd.newton_schulz(x, steps=steps, eps=eps).double()
    want, yard = ns(x.double(), steps, COEF, eps), ns(x.float(), steps, COEF, eps).double()
    for dim in (1, 0):
        size = want.norm(dim=dim)
        base = ((yard - want).norm(dim=dim) / (size + 1e-300)).max()
        tol = (8 * base + 2.0 ** -19 + (HALF_STEP[x.dtype] if x.dtype != torch.float32 else 0.0)) * size + floor_of(*x.shape, steps) + 1e-37
        off = (got - want).norm(dim=dim)
        assert bool((off <= tol).all()), (dim, float((off / tol).max()), float((off / (size + 1e-300)).max()))


SHAPES = [(40, 72), (50, 400), (64, 576), (700, 60), (100, 300), (600, 70), (512, 1500), (200, 9000), (1500, 2500)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("small", [1e-2, 1e-4, 1e-6, 1e-8])
def test_rows_and_columns_of_different_sizes(m, n, small):
    x = noise(m, n, m + n)
    rows, cols, both = x.clone(), x.clone(), x.clone()
    rows[::2] *= small
    cols[:, 1::2] *= small
    both[::3] *= small
    both[:, ::2] *= small ** 0.5
    for v in (rows, cols, both):
        held_everywhere(v)


@pytest.mark.parametrize("m,n", SHAPES)
def test_small_rows_grow_over_many_steps(m, n):
    x = noise(m, n, 1)
    x[::2] *= 1e-6
    held_everywhere(x, steps=12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_matrices_far_below_eps(m, n, dtype):
    """X_0 = X / (|X| + eps) is as small as X against eps, and grows by a^steps."""
    x = noise(m, n, m * n)
    x = x / x.double().norm().float()
    for size in (1e-7, 1e-10, 1e-13, 1e-16, 1e-20, 1e-30):
        held_everywhere((x * size).to(dtype))
    held_everywhere((x * 1e-15).to(dtype), steps=14)
    held_everywhere((x * 1e-3).to(dtype), eps=1.0)
    held_everywhere((x * 1e-9).to(dtype), eps=1e9, steps=20)


def test_small_and_large_matrices_of_one_call():
    xs = [noise(m, n, i) * s for i, ((m, n), s) in enumerate([((96, 300), 1.0), ((300, 96), 1e-18), ((64, 64), 1e-28), ((512, 1500), 1e12)])]
    out = dvae_amd.newton_schulz(xs)
    for x, y in zip(xs, out):
        want, yard = ns(x.double()), ns(x)
        assert float((y.double() - want).norm()) <= 8 * float((yard.double() - want).norm()) + 2.0 ** -19 * float(want.norm())


def test_muon_step_of_a_gradient_far_below_eps():
    """The step itself: a gradient of 1e-18, a learning rate that makes the update visible, from a parameter of zeros."""
    for shape in ((64, 90), (200, 300)):
        g = noise(*shape, 2) * 1e-18
        p, m = torch.zeros_like(g), torch.zeros_like(g)
        dvae_amd.muon_step([p], [g], [m], lr=1e9, momentum=0.0)
        s = max(1.0, shape[0] / shape[1]) ** 0.5
        want = -1e9 * s * ns(g.double())
        yard = -1e9 * s * ns(g).double()
        assert float((p.double() - want).norm()) <= 8 * float((yard - want).norm()) + 2.0 ** -19 * float(want.norm())


SMALL, BATCHED = (40, 72), (100, 300)


@pytest.mark.parametrize("eps", [0.0, 1e-320, 1e-7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [SMALL, (72, 40), (60, 700), BATCHED, (300, 100)])
def test_zero_matrix_comes_out_as_zeros(shape, dtype, eps):
    """Whatever eps is: 0 / (0 + 0) is not taken.  The other matrix of the call is orthogonalised as ever."""
    z, x = torch.zeros(shape, dtype=dtype, device="cuda"), noise(*shape, 5).to(dtype)
    out = dvae_amd.newton_schulz([z, x], eps=eps)
    assert not out[0].any() and torch.equal(out[1], dvae_amd.newton_schulz([x, x], eps=eps)[0])
    if dtype == torch.float32:
        p, m = torch.full(shape, 0.5, device="cuda"), torch.zeros(shape, device="cuda")
        dvae_amd.muon_step([p], [z], [m], eps=eps, weight_decay=0.0)
        assert bool((p == 0.5).all()) and not m.any()


@pytest.mark.parametrize("eps", [0.0, 1e-7])
@pytest.mark.parametrize("shape", [(1, 1), (5, 1), SMALL, (72, 40), (60, 700), BATCHED])
def test_non_finite_matrices_stay_to_themselves(shape, eps):
    """In the one-launch kernel as in the batched ones: NaNs all over, and nothing in the other matrices of the call."""
    good = noise(*shape, 6)
    nan, inf, both = good.clone(), good.clone(), good.clone()
    nan[-1, 0], inf[0, -1] = float("nan"), float("-inf")
    both[0, 0], both[-1, -1] = float("inf"), float("nan")
    ref = dvae_amd.newton_schulz([good] * 5, eps=eps)[0]
    out = dvae_amd.newton_schulz([nan, good, inf, good, both], eps=eps)
    assert all(bool(out[i].isnan().all()) for i in (0, 2, 4))
    assert torch.equal(out[1], ref) and torch.equal(out[3], ref)


@pytest.mark.parametrize("shape", [BATCHED, (300, 100), (1100, 640)])
def test_scale_of_the_input_in_the_batched_kernels(shape):
    x = noise(*shape, 7) * 1e-3
    ref = dvae_amd.newton_schulz(x)
    for s in (1e25, 1e38 / float(x.abs().max()), 1.0):
        y = dvae_amd.newton_schulz((x.double() * s).float())        # the factor itself leaves float32
        # |x| + eps is 2e-7 of itself away from |x|, which 1e-7 of a step's slope at most makes of the result, beside the roundings
        assert float((y - ref).norm()) <= 1e-4 * float(ref.norm())
    held_everywhere(x * 1e-30, eps=1e-28)
