"""Layer norm on libdvae_hip against its definition in 64 bits: forward, gradients, layouts, edges, streams, graphs."""
import pytest
import torch

import dvae_amd
from dvae_amd import _lib as L
from util_learn import ln_bound, ln_exact, ln_exact_grad, ln_grad_bounds

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def make(rows, c, dtype, seed=0, offset=1.0, affine=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=g) * (torch.rand(rows, 1, generator=g) + 0.5) + offset * torch.randn(rows, 1, generator=g))
    dy = torch.randn(rows, c, generator=g)
    w = 1 + 0.3 * torch.randn(c, generator=g) if affine else None
    b = 0.2 * torch.randn(c, generator=g) if affine else None
    return x.to(dtype).cuda(), dy.to(dtype).cuda(), None if w is None else w.cuda(), None if b is None else b.cuda()


def held(got, want, tol):
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= tol).all()), (float((d / tol).max()), float(d.max()))


def check(x, dy, w, b, eps=1e-5, xin=None, dyin=None):
    """x, dy: contiguous values; xin / dyin: the same values in the layout under test."""
    leaves = [(x if xin is None else xin).detach().requires_grad_(True)]
    leaves += [t.detach().clone().requires_grad_(True) if t is not None else None for t in (w, b)]
    y = dvae_amd.layer_norm(*leaves, eps)
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy if dyin is None else dyin)
    with torch.no_grad():
        assert torch.equal(dvae_amd.layer_norm(*leaves, eps), y)
    rows, c = x.shape
    want, xh, inv = ln_exact(x, w, b, eps)
    dx, dw, db = ln_exact_grad(dy, xh, inv, w)
    tx, tw, tb = ln_grad_bounds(x, dy, dx, xh, inv, w, c, rows)
    y2 = y.detach().reshape(rows, c)
    assert y.dtype == x.dtype and got[0].dtype == x.dtype
    held(y2, want, ln_bound(x, want, xh, inv, w, b, c))
    held(got[0].reshape(rows, c), dx, tx)
    if w is not None:
        held(got[1], dw, tw)
    if b is not None:
        held(got[-1], db, tb)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 2), (1, 512), (5, 7), (17, 31), (64, 16), (33, 32), (130, 64), (9, 65), (257, 128),
                                    (70, 193), (21, 256), (19, 300), (40, 512), (11, 513), (13, 777), (6, 1000), (37, 1024),
                                    (5, 1025), (3, 2048), (9, 2500), (4, 4096), (2, 4097), (3, 8192), (2, 8200), (2, 16384),
                                    (2, 16385), (3, 40001)])
def test_values_and_gradients(rows, c, dtype):
    check(*make(rows, c, dtype, seed=rows + c))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(40000, 24), (20011, 128), (9001, 515), (2100, 1536), (70, 20000)])
def test_many_rows(rows, c, dtype):
    check(*make(rows, c, dtype, seed=3))


@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
def test_optional_parameters(affine):
    x, dy, w, b = make(50, 96, torch.float32)
    check(x, dy, w if affine in ("both", "weight") else None, b if affine in ("both", "bias") else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0.0, 100.0])
def test_mean_far_from_zero(dtype, offset):
    """E[x^2] - E[x]^2 would lose the variance here; squared distances from the mean keep it."""
    x, dy, w, b = make(40, 384, dtype, offset=offset)
    check(x, dy, w, b)


def test_constant_rows_and_zero_rows():
    x = torch.cat([torch.zeros(2, 40), torch.full((2, 40), 2.0)]).cuda()      # 40 * 2 sums exactly: the variance is 0
    _, dy, w, b = make(4, 40, torch.float32)
    y = dvae_amd.layer_norm(x, w, b)
    assert torch.equal(y, b.expand(4, 40))
    check(x, dy, w, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,wide,first", [(193, 256, 0), (100, 128, 5), (31, 33, 1), (1500, 2048, 3), (17000, 17001, 1)])
def test_rows_inside_wider_ones(c, wide, first, dtype):
    rows = 23
    x, dy, w, b = make(rows, c, dtype, seed=c)
    xin, dyin = (torch.full((rows, wide), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    xin, dyin = xin[:, first:first + c], dyin[:, first:first + c]
    xin.copy_(x)
    dyin.copy_(dy)
    check(x, dy, w, b, xin=xin, dyin=dyin)


def test_other_layouts():
    x, dy, w, b = make(60, 48, torch.float32)
    check(x, dy, w, b, xin=x.t().contiguous().t(), dyin=dy.t().contiguous().t())       # columns adjacent: copied
    x4 = x.reshape(3, 4, 5, 48)
    leaf = x4.permute(0, 3, 1, 2).contiguous(memory_format=torch.channels_last)        # NHWC memory, channels last by a view
    y = dvae_amd.layer_norm(leaf.permute(0, 2, 3, 1), w, b)
    assert torch.equal(y, dvae_amd.layer_norm(x4, w, b))
    row = x[:1]
    leaf = row.clone().requires_grad_(True)
    y = dvae_amd.layer_norm(leaf.expand(7, 48), w, b)                                   # row stride 0
    g, = torch.autograd.grad(y, leaf, torch.ones((), device="cuda").expand(7, 48) * dy[:7])
    one = ln_exact(row, w, b, 1e-5)
    dxs = [ln_exact_grad(dy[i:i + 1], one[1], one[2], w)[0] for i in range(7)]
    assert float((g - sum(dxs)).abs().max()) <= 1e-4 * float(sum(d.abs() for d in dxs).max())
    leaf = x.clone().requires_grad_(True)
    dvae_amd.layer_norm(leaf, w, b).sum().backward()                                    # dy with strides 0, 0
    ones = torch.ones_like(x)
    _, xh, inv = ln_exact(x, w, b, 1e-5)
    dx = ln_exact_grad(ones, xh, inv, w)[0]
    held(leaf.grad, dx, ln_grad_bounds(x, ones, dx, xh, inv, w, 48, 60)[0])


def test_offsets_past_32_bits():
    """Rows 2^26 elements apart: the last ones start beyond 2^31 elements and 2^32 bytes."""
    rows, c, apart = 36, 200, 1 << 26
    x, dy, w, b = make(rows, c, torch.bfloat16)
    big = torch.empty(rows * apart, dtype=torch.bfloat16, device="cuda")
    xin = big.as_strided((rows, c), (apart, 1))
    dyin = big.as_strided((rows, c), (apart, 1), 1 << 20)
    xin.copy_(x)
    dyin.copy_(dy)
    check(x, dy, w, b, xin=xin, dyin=dyin)
    lib = L.lib()
    leaf = x.clone().requires_grad_(True)
    want = dvae_amd.layer_norm(leaf, w, b)
    out = big.as_strided((rows, c), (apart, 1), 2 << 20)
    L.check(lib.dvae_layer_norm_fwd(xin.data_ptr(), apart, w.data_ptr(), b.data_ptr(), out.data_ptr(), apart, None, None, rows, c, 1e-5,
                                    L.BF16, L.stream()))
    assert torch.equal(out, want)


def test_strided_parameters_and_another_gradient_type():
    x, dy, w, b = make(33, 72, torch.bfloat16)
    wide = torch.stack([w, b], 1).contiguous()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(dvae_amd.layer_norm(*leaves), leaves, dy)
    wide.requires_grad_(True)
    y = dvae_amd.layer_norm(leaves[0], wide[:, 0], wide[:, 1])
    g, = torch.autograd.grad(y, wide, dy.float())
    assert torch.equal(g[:, 0], ref[1]) and torch.equal(g[:, 1], ref[2])


def test_gradients_of_some_inputs_only():
    x, dy, w, b = make(33, 72, torch.bfloat16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = torch.autograd.grad(dvae_amd.layer_norm(*full), full, dy)
    for k in range(3):
        some = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        g, = torch.autograd.grad(dvae_amd.layer_norm(*some), some[k], dy)
        assert torch.equal(g, ref[k])


def test_gradient_against_differences():
    """Central differences of the 64-bit definition along random directions: the formula itself, not a copy of it."""
    x, dy, w, b = make(8, 40, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(dvae_amd.layer_norm(*leaves), leaves, dy)
    f = lambda *a: float((ln_exact(*a, 1e-5)[0] * dy.double()).sum())      # noqa: E731
    h = 1e-5
    for k in range(3):
        d = torch.randn(leaves[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64).cuda()
        lo, hi = [x.double(), w.double(), b.double()], [x.double(), w.double(), b.double()]
        lo[k], hi[k] = lo[k] - h * d, hi[k] + h * d
        slope = (f(*hi) - f(*lo)) / (2 * h)
        assert abs(float((got[k].double() * d).sum()) - slope) <= 1e-4 * float((got[k].double() * d).abs().sum())


def test_empty_and_leading_shapes():
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    y = dvae_amd.layer_norm(x, w, b)
    g = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 16, device="cuda"))
    assert y.shape == (0, 16) and g[0].shape == (0, 16) and not g[1].any() and not g[2].any()
    v = torch.randn(16, device="cuda")
    assert torch.equal(dvae_amd.layer_norm(v, w, b), dvae_amd.layer_norm(v[None], w, b)[0])
    assert dvae_amd.layer_norm(torch.zeros(2, 0, 16, device="cuda")).shape == (2, 0, 16)


def test_nan_and_infinity_stay_in_their_row():
    x, dy, w, b = make(12, 130, torch.float32)
    ref = dvae_amd.layer_norm(x, w, b)
    bad = x.clone()
    bad[3, 5], bad[7, 129] = float("nan"), float("inf")
    y = dvae_amd.layer_norm(bad, w, b)
    keep = [i for i in range(12) if i not in (3, 7)]
    assert torch.equal(y[keep], ref[keep]) and bool(y[3].isnan().all()) and bool(y[7, 129].isnan())


@pytest.mark.parametrize("c", [64, 193, 1500, 20000])
def test_a_row_does_not_depend_on_the_others(c):
    x, dy, w, b = make(300, c, torch.bfloat16)
    leaf = x.clone().requires_grad_(True)
    y = dvae_amd.layer_norm(leaf, w, b)
    dx, = torch.autograd.grad(y, leaf, dy)
    for lo, hi in ((0, 1), (17, 40), (299, 300)):
        part = x[lo:hi].clone().requires_grad_(True)
        z = dvae_amd.layer_norm(part, w, b)
        assert torch.equal(z, y[lo:hi]) and torch.equal(torch.autograd.grad(z, part, dy[lo:hi])[0], dx[lo:hi])


def test_c_entry_writes_nothing_else():
    """Strided outputs: the gaps between rows and the space around them keep their values."""
    rows, c, wide = 9, 37, 50
    lib = L.lib()
    x, dy, w, b = make(rows, c, torch.float32)
    buf = torch.full((rows * wide + 64,), 7.0, device="cuda")
    dbuf = buf.clone()
    st = torch.empty(2, rows, device="cuda")
    L.check(lib.dvae_layer_norm_fwd(x.data_ptr(), c, w.data_ptr(), b.data_ptr(), buf.data_ptr() + 4 * 32, wide, st.data_ptr(),
                                    st.data_ptr() + 4 * rows, rows, c, 1e-5, L.F32, L.stream()))
    n = lib.dvae_layer_norm_workspace_bytes(rows, c, L.F32)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    L.check(lib.dvae_layer_norm_bwd(dy.data_ptr(), c, x.data_ptr(), c, w.data_ptr(), st.data_ptr(), st.data_ptr() + 4 * rows,
                                    dbuf.data_ptr() + 4 * 32, wide, None, None, ws.data_ptr(), n, rows, c, L.F32, L.stream()))
    leaf = x.clone().requires_grad_(True)
    y = dvae_amd.layer_norm(leaf, w, b)
    for got, want in ((buf, y.detach()), (dbuf, torch.autograd.grad(y, leaf, dy)[0])):
        body = got[32:32 + rows * wide].view(rows, wide)
        assert torch.equal(body[:, :c], want) and bool((body[:, c:] == 7).all())
        assert bool((got[:32] == 7).all()) and bool((got[32 + rows * wide:] == 7).all())


def test_side_stream_and_module():
    x, dy, w, b = make(200, 256, torch.bfloat16)
    m = dvae_amd.LayerNorm(256).cuda()
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"weight": (256,), "bias": (256,)}
    ref = m(x)
    ref.backward(dy)
    grads = [m.weight.grad.clone(), m.bias.grad.clone()]
    m.zero_grad()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = m(x)
        g = torch.autograd.grad(y, (m.weight, m.bias), dy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ref) and torch.equal(g[0], grads[0]) and torch.equal(g[1], grads[1])
    assert dvae_amd.LayerNorm(8, affine=False).state_dict() == {}


def test_captured_forward_and_backward_replay():
    x, dy, w, b = make(500, 200, torch.float32)
    sx, sdy = x.clone().requires_grad_(True), dy.clone()
    sw, sb = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(dvae_amd.layer_norm(sx, sw, sb), (sx, sw, sb), sdy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dvae_amd.layer_norm(sx, sw, sb)
        out = [y, *torch.autograd.grad(y, (sx, sw, sb), sdy)]
    for seed in range(4):
        x, dy, w, b = make(500, 200, torch.float32, seed=10 + seed)
        with torch.no_grad():
            for d, s in ((sx, x), (sdy, dy), (sw, w), (sb, b)):
                d.copy_(s)
        graph.replay()
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        ref = dvae_amd.layer_norm(*leaves)
        want = [ref, *torch.autograd.grad(ref, leaves, dy)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_in_place_change_of_a_saved_input_is_noticed():
    x, dy, w, b = make(4, 16, torch.float32)
    leaf = x.clone().requires_grad_(True)
    mid = leaf * 1.0
    y = dvae_amd.layer_norm(mid, w, b)
    mid.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_refusals():
    x, dy, w, b = make(4, 16, torch.float32)
    for bad in (lambda: dvae_amd.layer_norm(x.half(), w, b), lambda: dvae_amd.layer_norm(x, w.bfloat16(), b),
                lambda: dvae_amd.layer_norm(x, w[:8], b), lambda: dvae_amd.layer_norm(x, w, b.cpu()),
                lambda: dvae_amd.layer_norm(x, w, b, -1.0), lambda: dvae_amd.layer_norm(x, w, b, float("nan")),
                lambda: dvae_amd.layer_norm(x[:, :0]), lambda: dvae_amd.layer_norm(x.sum()), lambda: dvae_amd.LayerNorm(8).cuda()(x)):
        with pytest.raises(RuntimeError):
            bad()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(dvae_amd.layer_norm(leaf, w, b).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
