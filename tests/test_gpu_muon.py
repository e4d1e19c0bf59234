"""Newton-Schulz orthogonalisation and the Muon step on libdvae_hip against their definitions in 64 bits."""
import math

import pytest
import torch

import dvae_amd
from dvae_amd import _lib as L
from dvae_amd import config as CFG
from util_learn import COEF, muon_expected, ns, ns_expected

pytestmark = pytest.mark.gpu


def matrix(m, n, seed=0, dtype=torch.float32, kind="noise"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g)
    if kind == "spiked":
        k = min(3, m, n)
        x = x + 4.0 / math.sqrt(max(m, n)) * torch.randn(m, k, generator=g) @ torch.randn(k, n, generator=g)
    return (1e-3 * x).to(dtype).cuda()


def held(got, x, **kw):
    want, tol = ns_expected(x, **kw)
    off = float((got.double().cpu() - want).norm())
    assert got.shape == want.shape and off <= tol, (tuple(x.shape), off / float(want.norm()), tol / float(want.norm()))


SHAPES = [(1, 1), (1, 2), (5, 1), (2, 2), (3, 288), (10, 2100), (27, 64), (64, 27), (31, 33), (63, 64), (64, 64), (64, 65), (65, 64),
          (64, 576), (576, 64), (96, 96), (127, 129), (128, 128), (129, 127), (128, 1152), (200, 130), (256, 300), (320, 700),
          (33, 512), (50, 257), (257, 20), (64, 768), (767, 63), (64, 769), (65, 768)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_orthogonalises(m, n, dtype):
    x = matrix(m, n, seed=m * 1000 + n, dtype=dtype)
    got = dvae_amd.newton_schulz(x)
    assert got.dtype == dtype and got.shape == x.shape
    held(got, x)


@pytest.mark.parametrize("m,n", [(640, 1100), (1100, 640), (1024, 1024), (2050, 130), (2112, 2112)])
def test_large(m, n):
    """Sizes whose products take the larger tiles, or that end inside one."""
    x = matrix(m, n, seed=5, kind="spiked")
    held(dvae_amd.newton_schulz(x), x)


def test_gradient_like_spectrum():
    x = matrix(128, 640, seed=2, kind="spiked")
    held(dvae_amd.newton_schulz(x), x)
    s = torch.linalg.svdvals(dvae_amd.newton_schulz(x).double().cpu())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 10])
def test_steps(steps):
    x = matrix(70, 100, seed=steps)
    held(dvae_amd.newton_schulz(x, steps=steps), x, steps=steps)


@pytest.mark.parametrize("coef", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (1.0, 0.0, 0.0)])
def test_other_coefficients(coef):
    x = matrix(80, 96, seed=4)
    held(dvae_amd.newton_schulz(x, steps=8, coefficients=coef), x, steps=8, coef=coef)


def test_list_of_any_shapes_is_each_alone():
    """One batch of launches for all: every matrix comes out as it does in a call of its own, up to how sums are cut."""
    shapes = SHAPES * 4                                       # more than one group of 64 jobs
    xs = [matrix(m, n, seed=i) for i, (m, n) in enumerate(shapes)]
    got = dvae_amd.newton_schulz(xs)
    assert isinstance(got, list) and len(got) == len(xs)
    for x, y in zip(xs, got):
        held(y, x)


@pytest.mark.parametrize("m,n,batch", [(16, 24, 33), (64, 64, 300), (9, 700, 40)])
def test_many_small_matrices(m, n, batch):
    g = torch.Generator().manual_seed(m)
    x = torch.randn(batch, m, n, generator=g).cuda()
    y = dvae_amd.newton_schulz(x)
    for i in {0, 1, 31, 32, batch // 2, batch - 1}:
        held(y[i], x[i])
        assert torch.equal(dvae_amd.newton_schulz(x[i]), y[i])


def test_batches_and_layouts():
    x = torch.stack([matrix(40, 72, seed=i) for i in range(6)])
    y = dvae_amd.newton_schulz(x)
    z = dvae_amd.newton_schulz(x.view(2, 3, 40, 72))
    assert z.shape == (2, 3, 40, 72) and torch.equal(z.view(6, 40, 72), y)
    for i in range(6):
        held(y[i], x[i])
    base = matrix(90, 200, seed=9)
    for v in (base.t(), base[10:50, 20:111], base[:, ::2], base[::3], base.t()[5:60:2], base[:1], base[:, :1], base[:, :1].t(),
              base[4].expand(30, 200)):
        held(dvae_amd.newton_schulz(v), v)
    held(dvae_amd.newton_schulz(torch.stack([base, base]).mT)[1], base.t())


def test_scale_of_the_input():
    """The norm is taken in 64 bits: neither large nor small values overflow it or vanish in it."""
    x = matrix(48, 80, seed=1)
    ref = dvae_amd.newton_schulz(x)
    for s in (1e25, 1e36, 1.0):
        y = dvae_amd.newton_schulz(x * s)
        assert float((y - ref).norm()) <= 1e-3 * float(ref.norm())
    tiny = x * 1e-30                                           # far under eps: what is left is the input over eps, a^5 as large
    held(dvae_amd.newton_schulz(tiny, eps=1e-28), tiny, eps=1e-28)


def test_zero_and_non_finite_matrices():
    good = matrix(70, 90, seed=3)
    ref = dvae_amd.newton_schulz([good, good])[0]
    zero, nan, inf = torch.zeros(70, 90, device="cuda"), good.clone(), good.clone()
    nan[5, 6], inf[69, 89] = float("nan"), float("-inf")
    out = dvae_amd.newton_schulz([zero, nan, good, inf])
    assert not out[0].any() and bool(out[1].isnan().all()) and bool(out[3].isnan().all())
    assert float((out[2] - ref).norm()) <= 2.0 ** -18 * float(ref.norm())
    part = good.clone()                                        # rows and columns of zeros stay zero
    part[10:20] = 0
    part[:, 5:9] = 0
    y = dvae_amd.newton_schulz(part)
    held(y, part)
    assert not y[10:20].any() and not y[:, 5:9].any()
    assert dvae_amd.newton_schulz([]) == [] and dvae_amd.newton_schulz(torch.zeros(3, 0, 4, device="cuda")).shape == (3, 0, 4)


def test_same_bits_every_time():
    xs = [matrix(m, n, seed=m) for m, n in ((64, 576), (128, 700), (300, 200), (10, 3000))]
    a, b = dvae_amd.newton_schulz(xs), dvae_amd.newton_schulz(xs)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_c_entry_writes_nothing_else():
    import array
    m, n, wide = 37, 53, 60
    x = matrix(m, n, seed=8)
    buf = torch.full((m * wide + 64,), 7.0, device="cuda")
    table = array.array("q", (x.data_ptr(), buf.data_ptr() + 4 * 32, 0, m, n, n, wide, 0))
    lib, at = L.lib(), table.buffer_info()[0]
    size = lib.dvae_newton_schulz_workspace_bytes(at, 1)
    ws = torch.full((size + 256,), 0x55, dtype=torch.uint8, device="cuda")
    coef = array.array("d", COEF)
    L.check(lib.dvae_newton_schulz(at, 1, coef.buffer_info()[0], 5, 1e-7, ws.data_ptr(), size, L.F32, L.stream()))
    body = buf[32:32 + m * wide].view(m, wide)
    assert torch.equal(body[:, :n], dvae_amd.newton_schulz(x)) and bool((body[:, n:] == 7).all())
    assert bool((buf[:32] == 7).all()) and bool((buf[32 + m * wide:] == 7).all()) and bool((ws[size:] == 0x55).all())


# ---- the Muon step --------------------------------------------------------------------------------------------------
def params_of(shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda s, k: (k * torch.randn(s, generator=g)).cuda()      # noqa: E731
    return [[r(s, k) for s in shapes] for k in (0.1, 1e-3, 1e-3)]


def step_held(shapes, seed=0, **kw):
    p, g, m = params_of(shapes, seed)
    want = [muon_expected(*t, **kw) for t in zip(p, g, m)]
    g0 = [t.clone() for t in g]
    dvae_amd.muon_step(p, g, m, **kw)
    for i, s in enumerate(shapes):
        p64, m64, tp, tm = want[i]
        dp, dm = float((p[i].double().cpu() - p64).norm()), float((m[i].double().cpu() - m64).norm())
        assert dp <= tp and dm <= tm, (s, dp, tp, dm, tm)
        assert torch.equal(g[i], g0[i])


MIXED = [(64, 3, 3, 3), (64,), (64, 64, 3, 3), (), (3,), (32, 3, 3, 3), (128, 64, 1, 1), (10, 700), (10,), (1, 5), (5, 1), (1,), (300, 20)]


@pytest.mark.parametrize("kw", [{}, {"nesterov": False}, {"momentum": 0.0}, {"weight_decay": 0.1, "lr": 0.3}, {"scale": "rms"},
                                {"steps": 3}, {"lr": 0.0, "weight_decay": 0.5}])
def test_step(kw):
    step_held(MIXED, **kw)


def test_many_parameters():
    step_held([(24, 5 + i % 40) if i % 3 else (i + 1,) for i in range(150)], seed=4)       # one launch for every 32 of them
    step_held([(24, 5 + i % 40) if i % 3 else (i + 1,) for i in range(149)] + [(70, 70)], seed=5)     # the batched phases
    step_held([(40, 3, 3, 3), (40000,), (9,)], seed=6)


@pytest.mark.parametrize("beside", [None, (80, 100)])      # alone in the one-launch kernel; among the batched phases
def test_c_entry_steps_every_row_of_a_vector(beside):
    import array
    shapes = [(3, 50)] + ([beside] if beside else [])
    p, g, m = params_of(shapes)
    mu, lr = 0.9, 0.1
    m64 = mu * m[0].double() + (1 - mu) * g[0].double()
    p64 = p[0].double() - lr * ((1 - mu) * g[0].double() + mu * m64)
    rows = [(g[i].data_ptr(), p[i].data_ptr(), m[i].data_ptr(), *s, s[1], s[1], int(i == 0)) for i, s in enumerate(shapes)]
    table, coef, lib = array.array("q", [v for r in rows for v in r]), array.array("d", COEF), L.lib()
    at = table.buffer_info()[0]
    size = lib.dvae_newton_schulz_workspace_bytes(at, len(rows))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    L.check(lib.dvae_muon_step(at, len(rows), lr, mu, 1, 0.0, L.MUON_SPECTRAL, coef.buffer_info()[0], 5, 1e-7, ws.data_ptr(), size,
                               L.stream()))
    # a handful of roundings of fp32 each: 2^-24 of the largest term, |p| or |m|
    assert float((m[0].double() - m64).abs().max()) <= 4 * 2.0 ** -24 * float(m64.abs().max() + g[0].abs().max())
    assert float((p[0].double() - p64).abs().max()) <= 4 * 2.0 ** -24 * float(p64.abs().max() + p[0].abs().max())


def test_vectors_only_and_views_of_a_bucket():
    step_held([(7,), (), (5000,)])
    shapes = [(3,), (33, 17), (64, 2, 3), (1,), (40, 41)]
    total = sum(math.prod(s) for s in shapes)
    bucket = [torch.full((total + 8,), 7.0, device="cuda") for _ in range(3)]
    src = params_of(shapes, seed=6)
    views = []
    for b, ts in zip(bucket, src):
        o, v = 3, []
        for t in ts:
            v.append(b[o:o + t.numel()].view(t.shape).copy_(t))
            o += t.numel()
        views.append(v)
    dvae_amd.muon_step(*views)
    dvae_amd.muon_step(*src)
    for v, t in zip(views[0] + views[2], src[0] + src[2]):
        assert torch.equal(v, t)
    assert all(bool((b[:3] == 7).all()) and bool((b[3 + total:] == 7).all()) for b in bucket)


def test_optimizer_matches_the_operator_and_resumes():
    def net(seed):
        torch.manual_seed(seed)
        return torch.nn.Sequential(torch.nn.Linear(48, 64), dvae_amd.LayerNorm(64), torch.nn.ReLU(), torch.nn.Linear(64, 10)).cuda()
    a, b = net(0), net(0)
    opt = CFG.from_dict({"optimizer": {"name": "FusedMuon", "lr": 0.05, "weight_decay": 0.01}}).optimizer(a.parameters())
    assert isinstance(opt, dvae_amd.FusedMuon)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    x, y = torch.randn(32, 48, device="cuda"), torch.randint(0, 10, (32,), device="cuda")
    mom = [torch.zeros_like(p) for p in b.parameters()]
    for k in range(3):
        for n in (a, b):
            n.zero_grad()
            torch.nn.functional.cross_entropy(n(x), y).backward()
        dvae_amd.muon_step(list(b.parameters()), [p.grad for p in b.parameters()], mom, lr=0.05 * 0.5 ** k, weight_decay=0.01)
        opt.step()
        sched.step()
        if k == 1:                                             # through a checkpoint
            sd = opt.state_dict()
            opt = dvae_amd.FusedMuon(a.parameters())
            opt.load_state_dict(sd)
            sched.optimizer = opt
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.equal(p, q)


def test_network_of_the_operators_takes_the_right_step():
    """Layer norm's gradients into the Muon step, as a training loop runs them: the gradients against 64-bit autograd on the
    CPU, the step against its definition on those gradients."""
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Linear(48, 64), dvae_amd.LayerNorm(64), torch.nn.Tanh(), torch.nn.Linear(64, 10)).cuda()
    ref = torch.nn.Sequential(torch.nn.Linear(48, 64), torch.nn.LayerNorm(64), torch.nn.Tanh(), torch.nn.Linear(64, 10)).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    x, y = torch.randn(32, 48), torch.randint(0, 10, (32,))
    torch.nn.functional.cross_entropy(net(x.cuda()), y.cuda()).backward()
    torch.nn.functional.cross_entropy(ref(x.double()), y).backward()
    opt = dvae_amd.FusedMuon(net.parameters(), lr=0.1)
    before = [p.detach().clone() for p in net.parameters()]
    grads = [p.grad.clone() for p in net.parameters()]
    versions = [p._version for p in net.parameters()]
    for g, r in zip(grads, ref.parameters()):
        # a gradient passes 48 + 64 + 32 term sums and a dozen elementwise roundings of terms no larger than a few times itself
        assert float((g.double().cpu() - r.grad).norm()) <= 512 * 2.0 ** -24 * float(r.grad.norm()) + 1e-9
    opt.step()
    for p, b, g, v in zip(net.parameters(), before, grads, versions):
        want, _, tol, _ = muon_expected(b, g, torch.zeros_like(b), lr=0.1)
        assert float((p.detach().double().cpu() - want).norm()) <= tol
        assert p._version > v


def test_classifier_trains_by_it():
    """The classifier's trunk notices the step (its packed weights are rebuilt) and runs on the stepped parameters."""
    torch.manual_seed(0)
    model = dvae_amd.ResNet18(10).cuda()
    opt = dvae_amd.FusedMuon(model.parameters(), lr=0.02)
    x, y = torch.rand(8, 3, 32, 32, device="cuda"), torch.arange(8, device="cuda")
    for _ in range(2):
        model.train()
        opt.zero_grad()
        torch.nn.functional.cross_entropy(model(x), y).backward()
        chosen = {n: (p.detach().clone(), p.grad.clone(), opt.state[p].get("momentum_buffer", torch.zeros_like(p)).clone())
                  for n, p in model.named_parameters() if n in ("conv1.weight", "layer1.0.conv1.weight", "layer2.0.shortcut.0.weight",
                                                                "bn1.weight", "linear.weight", "linear.bias")}
        opt.step()
        for n, p in model.named_parameters():
            if n in chosen:
                want, _, tol, _ = muon_expected(*chosen[n])
                assert float((p.detach().double().cpu() - want).norm()) <= tol, n
    model.eval()
    with torch.no_grad():
        out = model(x)
        model._engine.invalidate()
        assert torch.equal(out, model(x)) and bool(out.isfinite().all())


def test_dvae_trains_by_it():
    """The D-VAE's trainer with the optimiser a config names: parameters off the hot path have no gradient and stay."""
    torch.manual_seed(0)
    from dvae_amd import data as DD
    ds = DD.synthetic_cifar(n=128, seed=2)
    loaders = DD.DatasetGenerator(ds, train_batch_size=64, device="cuda").getDataLoader(train_shuffle=True, train_drop_last=True)
    model = dvae_amd.ResNet18DVAE(num_classes=10, stem_end_block=7, latent_dim=256)
    model.spatial_emb = True
    model.set_spatial_emb()
    model = model.cuda()
    opt = CFG.from_dict({"optimizer": {"name": "FusedMuon", "lr": 0.01}}).optimizer(model.parameters())

    class Cfg:
        grad_clip, log_frequency = 5.0, 100
    trainer = dvae_amd.VAE_Trainer(loaders, None, Cfg(), stage=0)
    model.train()
    off = model.layer3[0].conv1.weight.detach().clone()
    for images, labels in loaders["train_dataset"]:
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        old = {n: opt.state[p].get("momentum_buffer", torch.zeros_like(p)).clone() for n, p in model.named_parameters()}
        payload = trainer.train_batch(images, labels, model, None, opt, 0)
        assert math.isfinite(payload["loss"])
        for n, p in model.named_parameters():
            if n in ("conv1.weight", "decoder1.0.weight", "fc_mu.weight", "bn1.bias"):
                want, _, tol, _ = muon_expected(before[n], p.grad, old[n], lr=0.01)
                assert float((p.detach().double().cpu() - want).norm()) <= tol, n
    assert torch.equal(off, model.layer3[0].conv1.weight.detach())


def test_offsets_past_32_bits():
    """Rows 2^27 elements apart."""
    x = matrix(40, 60, seed=1)
    big = torch.empty(40 << 27, dtype=torch.float32, device="cuda")
    v = big.as_strided((40, 60), (1 << 27, 1))
    v.copy_(x)
    held(dvae_amd.newton_schulz(v), x)                          # too far apart for the one-launch kernel
    near = torch.zeros(40 << 22, dtype=torch.float32, device="cuda").as_strided((40, 60), (1 << 22, 1))
    near.copy_(x)
    assert torch.equal(dvae_amd.newton_schulz(near), dvae_amd.newton_schulz(x))
    y = matrix(66, 70, seed=2)                                  # through the batched kernels
    big = big[:(34 << 27)].view(-1)
    v = big.as_strided((66, 70), (1 << 26, 1))
    v.copy_(y)
    assert torch.equal(dvae_amd.newton_schulz(v), dvae_amd.newton_schulz(y))


def test_side_stream_and_captured_step():
    shapes = [(64, 9), (30, 200), (17,), (128, 128)]
    p, g, m = params_of(shapes)
    ref = [[t.clone() for t in ts] for ts in (p, g, m)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dvae_amd.muon_step(p, g, m)
    torch.cuda.current_stream().wait_stream(s)
    dvae_amd.muon_step(*ref)
    assert all(torch.equal(a, b) for a, b in zip(p + m, ref[0] + ref[2]))
    xs = [matrix(40, 60, seed=1), matrix(100, 30, seed=2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dvae_amd.muon_step(p, g, m)
        out = dvae_amd.newton_schulz(xs)
    for k in range(4):
        new = params_of(shapes, seed=20 + k)
        for d, t in zip(p + g + m, new[0] + new[1] + new[2]):
            d.copy_(t)
        for i, x in enumerate(xs):
            x.copy_(matrix(*x.shape, seed=30 + 2 * k + i))
        graph.replay()
        want = dvae_amd.newton_schulz([x.clone() for x in xs])
        dvae_amd.muon_step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p + m, new[0] + new[2])) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    """Every call has a workspace of its own: calls that overlap on two streams do not disturb each other."""
    xs = [matrix(256, 900, seed=i) for i in range(2)]
    ref = [dvae_amd.newton_schulz(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for s, x, o in zip(streams, xs, outs):
            with torch.cuda.stream(s):
                o.append(dvae_amd.newton_schulz(x))
    torch.cuda.synchronize()
    assert all(torch.equal(v, r) for o, r in zip(outs, ref) for v in o)


def test_refusals():
    x = matrix(8, 9)
    for bad in (lambda: dvae_amd.newton_schulz(x.half()), lambda: dvae_amd.newton_schulz([x, x.bfloat16()]),
                lambda: dvae_amd.newton_schulz(x[0]), lambda: dvae_amd.newton_schulz(x, steps=0),
                lambda: dvae_amd.newton_schulz(x, eps=-1.0), lambda: dvae_amd.newton_schulz(x, coefficients=(1.0, 2.0)),
                lambda: dvae_amd.newton_schulz(x, coefficients=(9.0, 0.0, 0.0)), lambda: dvae_amd.newton_schulz([x, x.cpu()]),
                lambda: dvae_amd.newton_schulz(x, coefficients=(float("nan"), 0.0, 0.0)),
                lambda: dvae_amd.newton_schulz(x.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError):
            bad()
    p, g, m = params_of([(8, 9), (4,)])
    for bad in (lambda: dvae_amd.muon_step(p, g[:1], m), lambda: dvae_amd.muon_step(p, g, m, scale="none"),
                lambda: dvae_amd.muon_step(p, g, m, momentum=1.0), lambda: dvae_amd.muon_step(p, g, m, lr=float("nan")),
                lambda: dvae_amd.muon_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0]]), lambda: dvae_amd.muon_step(p, m, m),
                lambda: dvae_amd.muon_step([p[0].t()], [g[0].t()], [m[0].t()]), lambda: dvae_amd.muon_step(p, g, [t.double() for t in m]),
                lambda: dvae_amd.muon_step([p[0]], [g[0][:4]], [m[0]])):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(ValueError):
        dvae_amd.FusedMuon([torch.nn.Parameter(x)], lr=-1.0)
