"""Host side of layer norm, Newton-Schulz and the Muon step: what the entry points refuse, and workspace sizes (no GPU)."""
from array import array

import pytest
import torch

import dvae_amd
from dvae_amd import _lib as L
from util_learn import COEF, ns

F = 1 << 20          # stands for a device address: nothing here gets as far as a launch


def table(*rows):
    return array("q", [v for r in rows for v in r])


def test_layer_norm_refuses_bad_arguments():
    lib = L.lib()
    fwd = lambda x=F, xs=8, y=F, ys=8, mean=None, inv=None, rows=4, c=8, eps=1e-5, dt=L.F32: lib.dvae_layer_norm_fwd(   # noqa: E731
        x, xs, None, None, y, ys, mean, inv, rows, c, eps, dt, None)
    assert fwd(rows=0) == 0 and fwd(rows=0, x=None, y=None) == 0
    for bad in (dict(x=None), dict(y=None), dict(c=0), dict(c=-3), dict(rows=-1), dict(ys=7), dict(xs=-8), dict(x=F + 1), dict(y=F + 2),
                dict(mean=F), dict(inv=F), dict(eps=-1.0), dict(eps=float("nan"))):
        assert fwd(**bad) == -1 and b"layer_norm_fwd" in lib.dvae_last_error(), bad
    assert fwd(dt=7) == -2 and fwd(dt=L.BF16, y=F + 1) == -1
    bwd = lambda dy=F, x=F, st=F, dx=F, dw=F, ws=F, n=1 << 30, rows=4, c=8, xs=8: lib.dvae_layer_norm_bwd(              # noqa: E731
        dy, 8, x, xs, None, st, st, dx, 8, dw, None, ws, n, rows, c, L.F32, None)
    for bad in (dict(dy=None), dict(x=None), dict(st=None), dict(ws=None), dict(ws=F + 4), dict(rows=-2), dict(c=0)):
        assert bwd(**bad) == -1 and b"layer_norm_bwd" in lib.dvae_last_error(), bad
    assert bwd(n=63) == -4 and bwd(dx=None, dw=None, ws=None, n=0) == 0
    for rows, c in ((0, 8), (1, 8), (10 ** 9, 8), (4, 40000), (10 ** 6, 1024)):
        n = lib.dvae_layer_norm_workspace_bytes(rows, c, L.F32)
        assert 0 < n <= 2 * 4 * c * 1024
    assert lib.dvae_layer_norm_workspace_bytes(-1, 8, L.F32) == 0 and lib.dvae_layer_norm_workspace_bytes(4, 0, L.F32) == 0


def test_layer_norm_refuses_rows_of_which_two_leave_32_bits():
    lib, c = L.lib(), 1 << 30
    assert lib.dvae_layer_norm_fwd(F, c, None, None, F, c, None, None, 1, c, 1e-5, L.F32, None) == -1
    assert lib.dvae_layer_norm_bwd(F, c, F, c, None, F, F, F, c, F, None, F, 1 << 40, 1, c, L.F32, None) == -1
    assert lib.dvae_layer_norm_workspace_bytes(1, c, L.F32) == 0 and lib.dvae_layer_norm_workspace_bytes(1, c - 1, L.F32) >= 8 * (c - 1)


def test_newton_schulz_and_muon_refuse_bad_arguments():
    lib = L.lib()
    good = (F, F, F, 6, 8, 8, 8, 0)

    def call(row=good, coef=COEF, steps=5, eps=1e-7, ws=F, n=1 << 40, dt=L.F32, count=1):
        t, c = table(row), array("d", coef)
        return lib.dvae_newton_schulz(t.buffer_info()[0], count, c.buffer_info()[0], steps, eps, ws, n, dt, None)

    def with_(i, v):
        return good[:i] + (v,) + good[i + 1:]
    assert call(count=0) == 0
    for bad in (dict(row=with_(0, 0)), dict(row=with_(1, 0)), dict(row=with_(3, 0)), dict(row=with_(4, -1)), dict(row=with_(5, -8)),
                dict(row=with_(6, 7)), dict(row=with_(7, 1)), dict(row=with_(3, 1 << 31)), dict(row=(F, F, F, 1 << 20, 1 << 12, 1 << 12, 1 << 12, 0)),
                dict(row=with_(0, F + 2)), dict(steps=0), dict(steps=101), dict(eps=-1e-9), dict(eps=float("inf")), dict(ws=None),
                dict(ws=F + 64), dict(count=-1), dict(coef=(9.0, 0, 0)), dict(coef=(3.0, 0, 0)), dict(coef=(1.0, 5.0, 0)),
                dict(coef=(float("nan"), 0, 0))):
        assert call(**bad) == -1 and b"newton_schulz" in lib.dvae_last_error(), bad
    assert call(n=100) == -4 and call(dt=3) == -2 and call(row=(F, F, F, 65, 65, 65, 65, 0), n=1024) == -4

    def muon(row=good, lr=0.1, mu=0.9, wd=0.0, rule=0, n=1 << 40):
        t, c = table(row), array("d", COEF)
        return lib.dvae_muon_step(t.buffer_info()[0], 1, lr, mu, 1, wd, rule, c.buffer_info()[0], 5, 1e-7, F, n, None)
    for bad in (dict(row=with_(2, 0)), dict(row=with_(5, 9)), dict(row=with_(6, 9)), dict(lr=-1.0), dict(lr=float("nan")), dict(mu=1.0),
                dict(mu=-0.1), dict(wd=-1.0), dict(rule=2)):
        assert muon(**bad) == -1 and b"muon_step" in lib.dvae_last_error(), bad
    assert muon(n=100) == -4


def test_newton_schulz_workspace_grows_with_the_list():
    lib = L.lib()
    rows = [(F, F, 0, 64, 576, 576, 576, 0), (F, F, 0, 512, 4608, 4608, 4608, 0), (F, F, 0, 1, 1, 1, 1, 0)]
    sizes = []
    for k in range(4):
        t = table(*rows[:k])
        sizes.append(lib.dvae_newton_schulz_workspace_bytes(t.buffer_info()[0], k))
    assert sizes == sorted(sizes) and sizes[2] >= 4 * 3 * 512 * 4608
    bad = table((F, F, 0, 0, 5, 5, 5, 0))
    assert lib.dvae_newton_schulz_workspace_bytes(bad.buffer_info()[0], 1) == 0
    assert lib.dvae_newton_schulz_workspace_bytes(None, 1) == 0


@pytest.mark.parametrize("coef,steps,fits", [(COEF, 5, True), (COEF, 100, True), ((1.5, -0.5, 0.0), 30, True), ((1.875, -1.25, 0.375), 30, True),
                                             ((2.0, 0.0, 0.0), 1, True), ((2.0, 0.0, 0.0), 2, False), ((7.5, -10.0, 4.0), 1, False)])
def test_coefficients_are_held_to_the_range(coef, steps, fits):
    """What the entry accepts keeps every iterate's singular values at 2 or below, by sampling the polynomial."""
    s = torch.linspace(0, 1, 20001, dtype=torch.float64)
    worst_x, worst_q = 0.0, 0.0
    for _ in range(steps):
        q = coef[0] + coef[1] * s ** 2 + coef[2] * s ** 4
        worst_q, s = max(worst_q, float(q.abs().max())), (s * q).abs()
        worst_x = max(worst_x, float(s.max()))
    t, c = table((F, F, 0, 6, 8, 8, 8, 0)), array("d", coef)
    rc = L.lib().dvae_newton_schulz(t.buffer_info()[0], 1, c.buffer_info()[0], steps, 1e-7, F, 16, L.F32, None)
    assert rc == (-4 if fits else -1)                   # -4: everything but the workspace was accepted
    assert (worst_x <= 2.0 and worst_q <= 7.0) == fits


def test_python_entries_refuse_host_tensors():
    x = torch.randn(4, 8)
    for call in (lambda: dvae_amd.layer_norm(x), lambda: dvae_amd.newton_schulz(x), lambda: dvae_amd.muon_step([x], [x], [x.clone()]),
                 lambda: dvae_amd.LayerNorm(8)(x)):
        with pytest.raises(RuntimeError, match="libdvae_hip|device"):
            call()
    assert dvae_amd.newton_schulz([]) == []
    dvae_amd.muon_step([], [], [])
    assert dvae_amd.FusedMuon([torch.nn.Parameter(x)]).step() is None          # no gradient: nothing to do


def test_oracle_of_the_iteration_acts_on_singular_values():
    """The tests' own 64-bit form: X = U diag(s) V^T goes to U diag(phi(...phi(s / |s|))) V^T."""
    x = torch.randn(12, 20, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    u, s, v = torch.linalg.svd(x, full_matrices=False)
    s = s / (s.norm() + 1e-7)
    for _ in range(5):
        s = COEF[0] * s + COEF[1] * s ** 3 + COEF[2] * s ** 5
    assert torch.allclose(ns(x), (u * s) @ v, atol=1e-9)
    assert torch.allclose(ns(x.t().contiguous()), ((u * s) @ v).t(), atol=1e-9)
