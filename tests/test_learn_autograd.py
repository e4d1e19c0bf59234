"""What torch's differentiation may ask of layer norm and of the orthogonalising entries beyond first gradients: refused aloud,
never answered with a missing (that is, zero) derivative."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import dvae_amd

GPU = pytest.param("cuda", marks=pytest.mark.gpu)


@pytest.mark.parametrize("dev", ["cpu", GPU])
def test_forward_mode_is_refused(dev):
    x, w = torch.randn(4, 8, device=dev), torch.ones(8, device=dev)
    with fw.dual_level():
        d, dw = fw.make_dual(x, torch.randn_like(x)), fw.make_dual(w, torch.randn_like(w))
        for call in (lambda: dvae_amd.layer_norm(d, w), lambda: dvae_amd.layer_norm(x, dw), lambda: dvae_amd.layer_norm(x, w, dw),
                     lambda: dvae_amd.LayerNorm(8).to(dev)(d), lambda: dvae_amd.newton_schulz(d), lambda: dvae_amd.newton_schulz([x, d]),
                     lambda: dvae_amd.muon_step([x], [d], [x.clone()]), lambda: dvae_amd.muon_step([d], [x], [x.clone()])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: dvae_amd.layer_norm(t, w), (x,), (x,))


@pytest.mark.gpu
def test_values_inside_a_dual_level_are_served():
    x = torch.randn(4, 8, device="cuda")
    want = dvae_amd.layer_norm(x), dvae_amd.newton_schulz(x)
    with fw.dual_level():
        assert torch.equal(dvae_amd.layer_norm(x), want[0]) and torch.equal(dvae_amd.newton_schulz(x), want[1])


def _on_the_host(monkeypatch):
    """layer_norm's autograd node over plain torch arithmetic: what the node itself does needs no kernel."""
    from contextlib import nullcontext
    from dvae_amd import norm

    def forward(x, weight, bias, eps, save):
        mean, inv = x.mean(-1), (x.var(-1, unbiased=False) + eps).rsqrt()
        y = torch.nn.functional.layer_norm(x, x.shape[-1:], weight, bias, eps)
        return y, torch.stack([mean.reshape(-1), inv.reshape(-1)])

    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        inv = stats[1].reshape(x.shape[:-1] + (1,))
        xh = (x - stats[0].reshape(x.shape[:-1] + (1,))) * inv
        g = dy if weight is None else dy * weight
        dx = inv * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        want = ctx.needs_input_grad
        return dx if want[0] else None, (dy * xh).sum(0) if want[1] else None, dy.sum(0) if want[2] else None, None
    monkeypatch.setattr(norm, "_check", lambda *a: None)
    monkeypatch.setattr(norm, "_forward", forward)
    monkeypatch.setattr(norm, "_backward", backward)
    monkeypatch.setattr(norm.L, "on_device", lambda d: nullcontext())


@pytest.mark.parametrize("dev", ["cpu", GPU])
def test_second_derivatives_are_refused_in_every_form(dev, monkeypatch):
    if dev == "cpu":
        _on_the_host(monkeypatch)
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(s, generator=g).to(dev).requires_grad_(True) for s in ((5, 8), (8,), (8,), (5, 8)))
    grad = torch.autograd.grad
    first = grad(dvae_amd.layer_norm(x, w, b), (x, w, b), dy.detach())

    def penalty(y, of, k, seed=None):
        got = grad(y, of, seed, create_graph=True)[k]
        assert got.requires_grad
        got.square().sum().backward()
    for call in (lambda: penalty(dvae_amd.layer_norm(x).sum(), (x,), 0),                     # dy is a constant: only x is differentiated
                 lambda: penalty(dvae_amd.layer_norm(x, w, b).sum(), (x, w, b), 0), lambda: penalty(dvae_amd.layer_norm(x, w, b).sum(), (x, w, b), 1),
                 lambda: penalty(dvae_amd.layer_norm(x.detach(), w, b), (w, b), 0, dy), lambda: penalty(dvae_amd.layer_norm(x.detach(), w, b), (w, b), 1, dy),
                 lambda: penalty(dvae_amd.layer_norm(x, w.detach()).square().sum(), (x,), 0)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            call()
    # a graph that is kept without being differentiated again costs nothing and changes nothing
    kept = grad(dvae_amd.layer_norm(x, w, b), (x, w, b), dy.detach(), create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, kept)) and kept[0].requires_grad and not kept[2].requires_grad
    # the weight's gradient is a constant where neither x nor dy is differentiated
    assert not grad(dvae_amd.layer_norm(x.detach(), w, b), w, dy.detach(), create_graph=True)[0].requires_grad
