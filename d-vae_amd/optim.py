"""Fused clip_grad_norm_ + Adam over the engine's flat parameter bucket.

Replaces the pair ``torch.nn.utils.clip_grad_norm_(model.parameters(), grad_clip)`` +
``torch.optim.Adam.step()`` of /root/reference/main_vae_disentangle.py:210-211 (Adam lr 5e-3,
weight_decay 0: configs/cifar10/resnet18DVAE.yaml:21-23) with two launches of libdvae_hip.  It is a
``torch.optim.Optimizer`` so the reference's ``config_s.scheduler(optimizer)`` (CosineAnnealingLR) and
``optimizer.param_groups[0]['lr']`` keep working.  Parameters off the hot path never receive a
gradient in the D-VAE stage (as in the reference, where Adam skips ``grad is None``) and are not touched.

Beside it, for any float32 parameters (the D-VAE's through autograd, the classifier's): ``FusedMuon``, whose step moves a
matrix by its momentum's nearest orthogonal matrix instead of the momentum itself, with ``muon_step`` and ``newton_schulz``,
the operators under it.  They have no counterpart in the reference.
"""
from array import array
import math

import torch

from . import _lib as L

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_SCALES = {"spectral": L.MUON_SPECTRAL, "rms": L.MUON_RMS}


def _workspace(table, count, device):
    n = L.lib().dvae_newton_schulz_workspace_bytes(table, count)
    return torch.empty(n, dtype=torch.uint8, device=device), n


def newton_schulz(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Orthogonalises matrices: X / (|X|_F + eps), then ``steps`` times X <- a X + (b A + c A^2) X with A = X X^T and
    (a, b, c) = ``coefficients``, which drives every singular value towards 1 and leaves the singular vectors.

    ``x``: a float32 or bfloat16 device tensor of shape [..., m, n], or a list of them of one type (any shapes: the whole list
    is one batch of launches, 65536 matrices at most).  Returns the same, in x's type and layout.  The products have float32
    accuracy for either type, as far as parts of a matrix go that are not below about 1e-7 of the rest (a row or column of
    1e-8 of the others' size comes out to 1e-5 of itself).  The result is not differentiable."""
    many = isinstance(x, (list, tuple))
    xs = list(x) if many else [x]
    L.refuse_tangents("newton_schulz", *xs)
    outs, table, keep = [], array("q"), []
    for i, t in enumerate(xs):
        if not t.is_cuda:
            raise RuntimeError("newton_schulz runs on libdvae_hip: it takes device tensors")
        if t.dtype not in (torch.float32, torch.bfloat16) or t.dtype != xs[0].dtype or t.device != xs[0].device:
            raise RuntimeError(f"newton_schulz: tensor {i} is {t.dtype} on {t.device}; all have to be float32 or all bfloat16, "
                               "on one device")
        if t.dim() < 2:
            raise RuntimeError(f"newton_schulz: tensor {i} of shape {tuple(t.shape)} is no matrix")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("newton_schulz is not differentiable: pass a detached tensor or call it under torch.no_grad()")
        m, n = t.shape[-2:]
        if t.numel() == 0:
            outs.append(torch.empty(t.shape, dtype=t.dtype, device=t.device))
            continue
        flat = t.detach()
        flip = not (flat.stride(-1) == 1 or n == 1) and (flat.stride(-2) == 1 or m == 1)
        if flip:                                     # stored by columns: the transpose is what lies in memory
            flat, m, n = flat.mT, n, m
        flat = flat.reshape(-1, m, n)
        if not (flat.stride(2) == 1 or n == 1):
            flat = flat.contiguous()
        keep.append(flat)
        out = torch.empty(t.shape[:-2] + (m, n), dtype=t.dtype, device=t.device)
        outs.append(out.mT if flip else out)
        size, src, dst = t.element_size(), flat.data_ptr(), out.data_ptr()
        step = flat.stride(0) * size
        stride = flat.stride(1)
        for b in range(flat.shape[0]):
            table.extend((src + b * step, dst + b * m * n * size, 0, m, n, stride, n, 0))
    count = len(table) // 8
    if count:
        device = xs[0].device
        with L.on_device(device):
            at = table.buffer_info()[0]
            ws, size = _workspace(at, count, device)
            coef = array("d", coefficients)
            if len(coef) != 3:
                raise RuntimeError(f"newton_schulz: three coefficients, got {len(coef)}")
            L.check(L.lib().dvae_newton_schulz(at, count, coef.buffer_info()[0], int(steps), float(eps), ws.data_ptr(), size,
                                               L.F32 if xs[0].dtype == torch.float32 else L.BF16, L.stream()))
    return outs if many else outs[0]


@torch.no_grad()
def muon_step(params, grads, momenta, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=COEFFICIENTS, eps=1e-7, scale="spectral"):
    """One Muon step, in place, over lists of contiguous float32 device tensors that share no memory:

        m <- momentum m + (1 - momentum) g;   u = (1 - momentum) g + momentum m  (nesterov; else m)
        p <- p (1 - lr weight_decay) - lr s newton_schulz(u)

    with every parameter of two or more dimensions taken as the matrix [shape[0], rest] and s = sqrt(max(1, rows / cols))
    (``scale="spectral"``) or 0.2 sqrt(max(rows, cols)) (``"rms"``: steps as long as Adam's).  Parameters of fewer dimensions
    (gains, biases) move by lr u.  All parameters go through the same two dozen launches."""
    if not len(params) == len(grads) == len(momenta):
        raise RuntimeError(f"muon_step: {len(params)} parameters, {len(grads)} gradients, {len(momenta)} momenta")
    L.refuse_tangents("muon_step", *params, *grads, *momenta)
    if scale not in _SCALES:
        raise RuntimeError(f"muon_step: scale {scale!r} ({sorted(_SCALES)})")
    table, written, read = array("q"), set(), set()
    device, f32 = params[0].device if params else None, torch.float32
    if device is not None and device.type != "cuda":
        raise RuntimeError("muon_step runs on libdvae_hip: it takes device tensors")
    for i, (p, g, m) in enumerate(zip(params, grads, momenta)):
        shape = p.shape
        if not (p.dtype == f32 and g.dtype == f32 and m.dtype == f32 and g.shape == shape and m.shape == shape and
                p.device == device and g.device == device and m.device == device and
                p.is_contiguous() and g.is_contiguous() and m.is_contiguous()):
            raise RuntimeError(f"muon_step: parameter, gradient and momentum {i} must be contiguous float32 tensors of one shape on "
                               f"{device}, got " + ", ".join(f"{t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}" for t in (p, g, m)))
        n = p.numel()
        if n == 0:
            continue
        pp, gp, mp = p.data_ptr(), g.data_ptr(), m.data_ptr()
        written.add(pp)
        written.add(mp)
        read.add(gp)
        if len(shape) < 2:
            table.extend((gp, pp, mp, 1, n, n, n, 1))
        else:
            cols = n // shape[0]
            table.extend((gp, pp, mp, shape[0], cols, cols, cols, 0))
    count = len(table) // 8
    if len(written) != 2 * count or not written.isdisjoint(read):
        raise RuntimeError("muon_step: a parameter or momentum is listed twice")
    if not count:
        return
    with L.on_device(device):
        at = table.buffer_info()[0]
        ws, size = _workspace(at, count, device)
        coef = array("d", coefficients)
        if len(coef) != 3:
            raise RuntimeError(f"muon_step: three coefficients, got {len(coef)}")
        L.check(L.lib().dvae_muon_step(at, count, float(lr), float(momentum), int(nesterov), float(weight_decay), _SCALES[scale],
                                       coef.buffer_info()[0], int(steps), float(eps), ws.data_ptr(), size, L.stream()))
    torch.autograd.graph.increment_version([*params, *momenta])     # packed weights and saved tensors notice the step


class FusedMuon(torch.optim.Optimizer):
    """Muon (K. Jordan and others, "Muon: an optimizer for hidden layers in neural networks", 2024) over ``muon_step``: a torch optimiser (schedulers, param groups, ``state_dict``) for contiguous float32 device
    parameters.  Parameters without a gradient are skipped.  Groups may differ in any option; each group is one batch of launches.  A step
    captured into a graph keeps the options it was captured with; the momenta have to exist before (one step outside the graph:
    made inside, every replay would clear them, so that is refused).  Its replays change the weights without their models'
    knowledge: ``model._engine.invalidate()`` before such a model's next eager call, as after writes through ``param.data``."""

    _OPTIONS = ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps", "scale")

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
                 eps=1e-7, scale="spectral"):
        if not (lr >= 0.0 and math.isfinite(lr)) or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError(f"FusedMuon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}")
        if scale not in _SCALES:
            raise ValueError(f"FusedMuon: scale {scale!r} ({sorted(_SCALES)})")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, scale=scale))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            momenta = []
            for p in params:
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if L.capturing(p.device):
                        raise RuntimeError("FusedMuon: the first step cannot be captured into a graph, whose replays would clear the "
                                           "momenta that it makes: take one step before the capture")
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                momenta.append(state["momentum_buffer"])
            muon_step(params, [p.grad.contiguous() for p in params], momenta, **{k: group[k] for k in self._OPTIONS})
        return loss


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, model, lr=5e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, max_norm=5.0):
        if weight_decay != 0.0:
            raise ValueError("the D-VAE configs use weight_decay 0; decay is not implemented in the fused kernel")
        self.model = model
        self.max_norm = max_norm
        self._pushed = None
        super().__init__(list(model.parameters()), dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def zero_grad(self, set_to_none: bool = True):
        # gradients live in the engine bucket and are overwritten by the next backward
        self.model._accumulate = False

    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0):
        eng = self.model._engine
        if eng is None:
            raise RuntimeError("FusedAdam.step() before any forward/backward on the GPU")
        g = self.param_groups[0]
        key = (id(eng), g["lr"], g["betas"], g["eps"], self.max_norm, grad_scale)
        if key != self._pushed:
            eng.set_hyper(lr=g["lr"], beta1=g["betas"][0], beta2=g["betas"][1], eps=g["eps"], max_norm=self.max_norm,
                          grad_scale=grad_scale)
            self._pushed = key
        eng.adam_step()
        self.model._accumulate = False
        return None
