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
