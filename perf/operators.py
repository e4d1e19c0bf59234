"""Cases of the layer-norm, Newton-Schulz and Muon operators: inputs, plain forms, 64-bit results and the work each needs.

``own`` is False: ``run`` computes an operator in elementary torch operations, in 32 bits (the Frobenius norm in 64).
``own`` is True: ``run`` makes the calls a user of the framework makes.

Operators ("op" of a case):
  ln_fwd    layer norm of inference: y
  ln_train  layer norm with gradients: y, dx, dweight, dbias
  ns        the quintic Newton-Schulz iteration that orthogonalises matrices: a tensor [..., m, n]
  muon      one optimiser step over a list of parameters that are views of flat buckets (parameters, gradients, momenta)
"""
import math

import torch

own = False

EPS_LN = 1e-5
EPS_NS = 1e-7
COEF = (3.4445, -4.7750, 2.0315)
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

# Parameters of the networks this repository trains, in the order of their buckets.
_DVAE = ("64x3x3x3 64 64 " + "64x64x3x3 64 64 " * 4 + "128x64x3x3 128 128 128x128x3x3 128 128 128x64x1x1 128 128 "
         "256x128x1x1 256x128x1x1 256 256 128x256x1x1 128 " + "128x64x4x4 64 64x64x3x3 64 64x32x3x3 32 32x3x3x3 3 " * 2 + "10x32768")
_RESNET18 = ("64x3x3x3 64 64 " + "64x64x3x3 64 64 " * 4 + "128x64x3x3 128 128 128x128x3x3 128 128 128x64x1x1 128 128 "
             + "128x128x3x3 128 128 " * 2 + "256x128x3x3 256 256 256x256x3x3 256 256 256x128x1x1 256 256 " + "256x256x3x3 256 256 " * 2
             + "512x256x3x3 512 512 512x512x3x3 512 512 512x256x1x1 512 512 " + "512x512x3x3 512 512 " * 2 + "10x512 10")


def listed():
    return [
        # one pooled feature vector of the classifier, as a served request brings it: latency
        {"name": "ln_token", "op": "ln_fwd", "rows": 1, "channels": 512, "stride": 512, "dtype": "f32"},
        # an odd number of channels inside the padded rows of an activation map
        {"name": "ln_padded_rows", "op": "ln_fwd", "rows": 10007, "channels": 193, "stride": 256, "dtype": "f32"},
        # every 16x16 map of a purification batch of 2048 images, 128 channels
        {"name": "ln_purify_batch", "op": "ln_fwd", "rows": 524288, "channels": 128, "stride": 128, "dtype": "bf16"},
        # a training batch of pooled features
        {"name": "ln_train_head", "op": "ln_train", "rows": 128, "channels": 512, "stride": 512, "dtype": "f32"},
        # an odd number of rows of a width that is no power of two
        {"name": "ln_train_odd", "op": "ln_train", "rows": 32749, "channels": 1000, "stride": 1000, "dtype": "f32"},
        # wide rows, many of them
        {"name": "ln_train_wide", "op": "ln_train", "rows": 16384, "channels": 4096, "stride": 4096, "dtype": "bf16"},
        # the first convolution's update: the smallest matrix of the networks, tall
        {"name": "ns_conv1", "op": "ns", "batch": 1, "m": 64, "n": 27, "dtype": "f32"},
        # the four 3x3 convolutions of layer1
        {"name": "ns_layer1", "op": "ns", "batch": 4, "m": 64, "n": 576, "dtype": "f32"},
        # a 3x3 convolution of layer4
        {"name": "ns_layer4", "op": "ns", "batch": 1, "m": 512, "n": 4608, "dtype": "bf16"},
        # a large square matrix
        {"name": "ns_square", "op": "ns", "batch": 1, "m": 2048, "n": 2048, "dtype": "f32"},
        # one step of the D-VAE's live parameters
        {"name": "muon_dvae", "op": "muon", "shapes": _DVAE},
        # one step of the classifier's parameters
        {"name": "muon_resnet18", "op": "muon", "shapes": _RESNET18},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_train", "ns", "muon"])
    if op in ("ln_fwd", "ln_train"):
        channels = _log(rng, 8, 8192)
        rows = _log(rng, 1, min(524288, (1 << 26) // channels))
        stride = channels if rng.random() < 0.7 else channels + _log(rng, 1, 64)
        return {"op": op, "rows": rows, "channels": channels, "stride": stride, "dtype": rng.choice(["f32", "bf16"])}
    if op == "ns":
        m, n = _log(rng, 8, 2048), _log(rng, 8, 4608)
        most = _flops([(2048, 2048)]) / _flops([(m, n)])
        batch = _log(rng, 1, 8) if most >= 8 else 1
        if most < 1:
            n = min(n, 2048)
        return {"op": op, "batch": batch, "m": m, "n": n, "dtype": rng.choice(["f32", "bf16"])}
    shapes = []
    for _ in range(_log(rng, 1, 40)):
        if rng.random() < 0.4:
            shapes.append(str(_log(rng, 3, 4096)))
        elif rng.random() < 0.5:
            shapes.append("%dx%d" % (_log(rng, 3, 512), _log(rng, 3, 2048)))
        else:
            shapes.append("%dx%dx%dx%d" % ((_log(rng, 3, 256), _log(rng, 3, 256)) + ((3, 3) if rng.random() < 0.8 else (1, 1))))
    return {"op": op, "shapes": " ".join(shapes)}


# ---- inputs --------------------------------------------------------------------------------------
def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def _matrix(shape):
    return shape[0], math.prod(shape[1:])


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _gradient(gen, batch, m, n):
    """What a matrix's gradient looks like: noise of the mini-batch and a few strong directions."""
    g = torch.randn(batch, m, n, device="cuda", generator=gen)
    k = min(4, m, n)
    u = torch.randn(batch, m, k, device="cuda", generator=gen)
    v = torch.randn(batch, k, n, device="cuda", generator=gen)
    return 1e-3 * (g + (2.0 / math.sqrt(max(m, n))) * (u @ v))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op in ("ln_fwd", "ln_train"):
        rows, c, stride = case["rows"], case["channels"], case["stride"]
        std = torch.rand(rows, 1, device="cuda", generator=gen) + 0.5
        x = torch.randn(rows, stride, device="cuda", generator=gen) * std + torch.randn(rows, 1, device="cuda", generator=gen)
        x = x.to(_dtype(case))[:, :c]
        s = {"case": case, "x": x,
             "w": 1.0 + 0.2 * torch.randn(c, device="cuda", generator=gen), "b": 0.1 * torch.randn(c, device="cuda", generator=gen)}
        if op == "ln_train":
            s["dy"] = (torch.randn(rows, c, device="cuda", generator=gen) * 0.1).to(_dtype(case))
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
        return s
    if op == "ns":
        return {"case": case, "x": _gradient(gen, case["batch"], case["m"], case["n"]).to(_dtype(case))}
    shapes = _shapes(case)
    total = sum(math.prod(s) for s in shapes)
    bucket = {k: torch.empty(total, device="cuda") for k in ("p", "g", "m")}
    views = {k: [] for k in bucket}
    o = 0
    for s in shapes:
        n = math.prod(s)
        for k in bucket:
            views[k].append(bucket[k][o:o + n].view(s))
        o += n
        if len(s) > 1:
            rows, cols = _matrix(s)
            grad, mom = _gradient(gen, 2, rows, cols).view((2,) + s)
        else:
            grad, mom = 1e-3 * torch.randn(2, n, device="cuda", generator=gen)
        views["g"][-1].copy_(grad)
        views["m"][-1].copy_(mom)
        views["p"][-1].copy_(torch.randn(s, device="cuda", generator=gen) * (2.0 / math.sqrt(n / s[0])))
    return {"case": case, "bucket": bucket, "views": views}


# ---- plain forms -----------------------------------------------------------------------------------
def _plain_layer_norm(x, w, b):
    xf = x.float()
    d = xf - xf.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS_LN)
    xh = d * r
    return (xh * w + b).to(x.dtype), xh, r


def _plain_layer_norm_grad(dy, xh, r, w, dtype):
    dyf = dy.float()
    g = dyf * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx.to(dtype), (dyf * xh).sum(0), dyf.sum(0)


def _plain_newton_schulz(x):
    a, b, c = COEF
    tall = x.shape[-2] > x.shape[-1]
    y = x.float()
    y = y.mT.contiguous() if tall else y
    norm = y.double().square().sum((-2, -1), keepdim=True).sqrt() + EPS_NS
    y = y / norm.float()
    for _ in range(5):
        s = y @ y.mT.contiguous()
        y = a * y + (b * s + c * (s @ s)) @ y
    return (y.mT if tall else y).to(x.dtype)


def _plain_muon(params, grads, momenta):
    for p, g, m in zip(params, grads, momenta):
        m.mul_(MOMENTUM).add_(g, alpha=1.0 - MOMENTUM)
        u = g * (1.0 - MOMENTUM) + m * MOMENTUM
        p.mul_(1.0 - LR * DECAY)
        if p.dim() < 2:
            p.sub_(u, alpha=LR)
        else:
            rows, cols = _matrix(p.shape)
            p.sub_(_plain_newton_schulz(u.view(rows, cols)).view(p.shape), alpha=LR * math.sqrt(max(1.0, rows / cols)))


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        import dvae_amd
        if op == "ln_fwd":
            return dvae_amd.layer_norm(state["x"], state["w"], state["b"], EPS_LN)
        if op == "ln_train":
            leaves = (state["x"], state["w"], state["b"])
            y = dvae_amd.layer_norm(*leaves, EPS_LN)
            return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
        if op == "ns":
            return dvae_amd.newton_schulz(state["x"])
        v = state["views"]
        dvae_amd.muon_step(v["p"], v["g"], v["m"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
        return [state["bucket"]["p"], state["bucket"]["m"]]
    with torch.no_grad():
        if op == "ln_fwd":
            return _plain_layer_norm(state["x"], state["w"], state["b"])[0]
        if op == "ln_train":
            y, xh, r = _plain_layer_norm(state["x"], state["w"], state["b"])
            return [y, *_plain_layer_norm_grad(state["dy"], xh, r, state["w"], state["x"].dtype)]
        if op == "ns":
            return _plain_newton_schulz(state["x"])
        v = state["views"]
        _plain_muon(v["p"], v["g"], v["m"])
        return [state["bucket"]["p"], state["bucket"]["m"]]


# ---- the definition in 64 bits -----------------------------------------------------------------------
def _exact_orthogonal(x):
    """X_k = T_k X_0 with T_k a polynomial of the Gram matrix G = X_0 X_0^T: T <- (a I + b H + c H^2) T, H = T G T."""
    if x.shape[0] > x.shape[1]:
        return _exact_orthogonal(x.t().contiguous()).t()
    a, b, c = COEF
    x = x / (torch.linalg.vector_norm(x) + EPS_NS)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    gram = torch.matmul(x, x.t())
    t = eye
    for _ in range(5):
        h = torch.matmul(torch.matmul(t, gram), t)
        t = torch.matmul(a * eye + torch.matmul(b * eye + c * h, h), t)
    return torch.matmul(t, x)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("ln_fwd", "ln_train"):
        with torch.no_grad():
            x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
            n = x.shape[1]
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            inv = (var + EPS_LN) ** -0.5
            xh = (x - mean) * inv
            y = torch.addcmul(b, xh, w)
            if op == "ln_fwd":
                return y
            dy = s["dy"].double()
            p1 = torch.mv(dy, w)[:, None]
            p2 = (dy * w * xh).sum(1, keepdim=True)
            dx = inv / n * (n * dy * w - p1 - xh * p2)
            return [y, dx, torch.linalg.vecdot(dy.t(), xh.t()), dy.sum(0)]
    if op == "ns":
        return torch.stack([_exact_orthogonal(v) for v in s["x"].double()])
    p, m = [], []
    for pp, g, mm in zip(*(s["views"][k] for k in ("p", "g", "m"))):
        pp, g, mm = pp.double(), g.double(), mm.double()
        mm = MOMENTUM * mm + (1.0 - MOMENTUM) * g
        u = (1.0 - MOMENTUM) * g + MOMENTUM * mm
        scale = 1.0
        if pp.dim() > 1:
            rows, cols = _matrix(pp.shape)
            u = _exact_orthogonal(u.reshape(rows, cols)).reshape(pp.shape)
            scale = max(1.0, rows / cols) ** 0.5
        p.append((pp * (1.0 - LR * DECAY) - LR * scale * u).reshape(-1))
        m.append(mm.reshape(-1))
    return [torch.cat(p), torch.cat(m)]


# ---- what a pass cannot do without --------------------------------------------------------------------
def _flops(matrices):
    """Five steps: X X^T and its square are symmetric (half of either), the third product is whole."""
    total = 0.0
    for m, n in matrices:
        p, q = min(m, n), max(m, n)
        total += 5.0 * (p * (p + 1.0) * q + p * (p + 1.0) * p + 2.0 * p * p * q)
    return total


def work(case):
    op = case["op"]
    if op in ("ln_fwd", "ln_train"):
        n, size = case["rows"] * case["channels"], 4 if case["dtype"] == "f32" else 2
        if op == "ln_fwd":
            return {"bytes": 2.0 * n * size + 8.0 * case["channels"], "flops": 8.0 * n}
        return {"bytes": 4.0 * n * size + 16.0 * case["channels"], "flops": 20.0 * n}
    if op == "ns":
        n, size = case["batch"] * case["m"] * case["n"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2.0 * n * size, "flops": _flops([(case["m"], case["n"])] * case["batch"])}
    shapes = _shapes(case)
    return {"bytes": 20.0 * sum(math.prod(s) for s in shapes), "flops": _flops([_matrix(s) for s in shapes if len(s) > 1])}
