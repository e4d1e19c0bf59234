"""``VAE_Trainer`` with a stock optimiser on two ranks (CPU, gloo): the step of the global batch, on every rank."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn as nn

from dvae_amd import dist as D
from dvae_amd.trainer import VAE_Trainer


class TinyVAE(nn.Module):
    """The model's call signature on plain torch layers, without per-batch statistics or noise: the gradients of a global batch
    are the mean of its samples'."""

    def __init__(self):
        super().__init__()
        self.enc, self.dec = nn.Conv2d(3, 4, 3, 2, 1), nn.ConvTranspose2d(2, 3, 4, 2, 1)
        self.per, self.unused = nn.Conv2d(3, 3, 1), nn.Linear(2, 2)

    def forward(self, x, y):
        mu, lv = self.enc(x).chunk(2, 1)
        return torch.zeros(x.shape[0], 10), self.dec(mu).sigmoid(), mu, lv, self.per(x)


class Config:
    grad_clip, log_frequency = 0.5, 100


def _batch():
    g = torch.Generator().manual_seed(1)
    x = torch.rand(8, 3, 8, 8, generator=g)
    x[4:] *= 3.0                        # the second rank's samples: other losses, on the other side of the gates
    return x, torch.arange(8) % 10


def _step(lo, hi, kd, epoch, optimizer):
    torch.manual_seed(0)
    model = TinyVAE()
    x, y = _batch()
    opt = optimizer(model.parameters())
    t = VAE_Trainer(None, None, Config(), stage=1, kd=kd, monitor_every=0)
    out = [t.train_batch(x[lo:hi], y[lo:hi], model, None, opt, epoch) for _ in range(3)]
    return model, out


def _sgd(p):
    return torch.optim.SGD(p, lr=0.5)


def _kld_of(lo, hi):
    torch.manual_seed(0)
    m = TinyVAE()
    x, y = _batch()
    _, _, mu, lv, _ = m(x[lo:hi], y[lo:hi])
    return float(torch.mean(-0.5 * torch.sum(1 + lv - mu ** 2 - lv.exp(), dim=1)).detach())


def _worker(rank, world, port, tmp, kd, epoch, cut):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    torch.set_num_threads(1)
    D.init_from_env("gloo")
    model, out = _step(*((0, cut) if rank == 0 else (cut, 8)), kd, epoch, _sgd)
    torch.save({"p": [p.detach() for p in model.parameters()], "out": out}, os.path.join(tmp, f"r{rank}.pt"))
    dist.destroy_process_group()


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


@pytest.mark.parametrize("gate,epoch,cut", [("open", 0, 4), ("between", 11, 4), ("shut", 11, 4), ("between", 0, 3)])
def test_generic_route_steps_the_global_batch(tmp_path, gate, epoch, cut):
    a, b, both = _kld_of(0, cut), _kld_of(cut, 8), _kld_of(0, 8)
    kd = {"open": 0.5 * min(a, b), "between": 0.5 * (both + min(a, b)), "shut": 2 * max(a, b)}[gate]
    mp.spawn(_worker, args=(2, _free_port(), str(tmp_path), kd, epoch, cut), nprocs=2, join=True)
    got = [torch.load(tmp_path / f"r{r}.pt", weights_only=True) for r in range(2)]
    want, out = _step(0, 8, kd, epoch, _sgd)
    for x, y in zip(got[0]["p"], got[1]["p"]):
        assert torch.equal(x, y)                                     # one model on all ranks, to the bit
    for x, y in zip(got[0]["p"], want.parameters()):
        assert torch.allclose(x, y.detach(), rtol=1e-5, atol=1e-6)   # some dozens of fp32 roundings of values of order one
    for k in ("loss", "loss_rec", "loss_rec_p", "kld_loss", "|gn|", "psnr"):
        for r in range(2):
            for o, w in zip(got[r]["out"], out):
                assert abs(o[k] - w[k]) <= 1e-5 * max(1.0, abs(w[k])), (k, o[k], w[k])


def test_ranks_draw_noise_of_their_own(monkeypatch):
    """The D-VAE's own noise, keyed by position: no index is drawn twice by the ranks of a call, or by two calls, and one
    process draws what it always drew."""
    import dvae_amd
    model = dvae_amd.ResNet18DVAE(num_classes=10, stem_end_block=7, latent_dim=256)
    seen = []
    for world in (1, 3):
        drawn = []
        for call in range(4):
            model._draws = call
            for rank in range(world):
                monkeypatch.setattr(D, "world_info", lambda rank=rank, world=world: (rank, world))
                first = model._first_draw(5)
                drawn += range(first, first + 5)
        assert sorted(drawn) == list(range(4 * world * 5))
        seen.append(drawn)
    assert seen[0] == list(range(20))
