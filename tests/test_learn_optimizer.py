"""FusedMuon and graphs: what a captured step may and may not hold."""
import pytest
import torch

import dvae_amd


def test_first_step_inside_a_capture_is_refused(monkeypatch):
    p = torch.nn.Parameter(torch.randn(4, 8))
    p.grad = torch.randn(4, 8)
    monkeypatch.setattr(dvae_amd._lib, "capturing", lambda device: True, raising=False)
    opt = dvae_amd.FusedMuon([p])
    with pytest.raises(RuntimeError, match="before the capture"):
        opt.step()
    assert not opt.state[p]


@pytest.mark.gpu
def test_captured_steps_keep_their_momentum():
    g = torch.Generator().manual_seed(0)
    shapes = [(24, 40), (70, 90), (24,)]
    start = [torch.randn(s, generator=g).cuda() for s in shapes]
    grads = [[torch.randn(s, generator=g).cuda() for s in shapes] for _ in range(6)]

    def made():
        ps = [torch.nn.Parameter(t.clone()) for t in start]
        for p, t in zip(ps, grads[0]):
            p.grad = t.clone()
        return ps, dvae_amd.FusedMuon(ps, lr=0.05)
    eager, opt_e = made()
    graphed, opt_g = made()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"), torch.cuda.graph(graph):
        opt_g.step()
    assert all(torch.equal(p, t) for p, t in zip(graphed, start))
    opt_e.step()
    opt_g.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt_g.step()
    for k in range(1, 6):
        for ps in (eager, graphed):
            for p, t in zip(ps, grads[k]):
                p.grad.copy_(t)
        opt_e.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, graphed):
            assert torch.equal(p, q)
            assert torch.equal(opt_e.state[p]["momentum_buffer"], opt_g.state[q]["momentum_buffer"])
