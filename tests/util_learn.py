"""64-bit forms of layer norm, the Newton-Schulz iteration and the Muon step, and the rounding bounds their tests use."""
import math

import torch

COEF = (3.4445, -4.7750, 2.0315)
U32 = 2.0 ** -24                                   # half a step of fp32, relative
HALF_STEP = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}


def ln_exact(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    inv = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * inv
    y = xh if w is None else xh * w.double()
    return (y if b is None else y + b.double()), xh, inv


def ln_exact_grad(dy, xh, inv, w):
    dy = dy.double()
    g = dy if w is None else dy * w.double()
    dx = inv * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def ln_depth(c):
    """Longest chain of additions a row's sum goes through: per thread at most max(16, C / 1024), then shuffles and waves."""
    return max(16, -(-c // 1024)) + 6 + 16


def ln_xhat_bound(x, xh, inv, c):
    """|computed xh - xh|: the mean is off by depth u mean|x|, x - mean by that and one rounding of it, the variance and the
    root by depth + 4 roundings relative (which multiply xh)."""
    d = ln_depth(c)
    off = d * U32 * x.double().abs().mean(-1, keepdim=True) * inv
    return 2 * off + (2 * off.square() + (d + 6) * U32) * xh.abs()


def ln_bound(x, y, xh, inv, w, b, c):
    """of y: xh's error times |w|, two roundings, and the rounding to y's type."""
    wa = 1.0 if w is None else w.double().abs()
    ba = 0.0 if b is None else b.double().abs()
    return ln_xhat_bound(x, xh, inv, c) * wa + 4 * U32 * (xh.abs() * wa + ba) + HALF_STEP[x.dtype] * y.abs() + 1e-38


def ln_grad_bounds(x, dy, dx, xh, inv, w, c, rows):
    """of dx, dw, db.  mean(g) and mean(g xh) are off by depth roundings of mean|g| and mean|g xh| and by xh's error; a column
    sum goes through at most rows + 64 additions."""
    d = ln_depth(c)
    e = ln_xhat_bound(x, xh, inv, c)
    dya = dy.double().abs()
    g = dya if w is None else dya * w.double().abs()
    m1, m2, me = (t.mean(-1, keepdim=True) for t in (g, g * xh.abs(), g * e))
    inner = (d + 4) * U32 * (g + m1 + 2 * xh.abs() * m2) + e * m2 + xh.abs() * me
    tol_x = inv * inner + (d + 8) * U32 * inv * (g + m1 + xh.abs() * m2) + HALF_STEP[x.dtype] * dx.abs() + 1e-38
    chain = min(rows, 64) + math.sqrt(max(rows, 1)) + 64      # the longest order in use: rows over the workgroups, then the slabs
    tol_w = (dya * e).sum(0) + chain * U32 * (dya * (xh.abs() + e)).sum(0) + 1e-38
    tol_b = chain * U32 * dya.sum(0) + 1e-38
    return tol_x, tol_w, tol_b


def ns(x, steps=5, coef=COEF, eps=1e-7):
    """The definition, in x's own precision (float64 for the expected value, float32 for the yardstick)."""
    a, b, c = coef
    if x.shape[0] > x.shape[1]:
        return ns(x.t().contiguous(), steps, coef, eps).t()
    x = x / (x.double().square().sum().sqrt() + eps).to(x.dtype)
    for _ in range(steps):
        g = x @ x.t().contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def ns_expected(x, steps=5, coef=COEF, eps=1e-7):
    """Expected value and its tolerance in the Frobenius norm.  Operands carry 22 bits against fp32's 24, so a product's input
    error is at most four times fp32's, and the sums are as long: eight times the error of the same iteration in float32,
    plus 2^-20 where that happens to be exact, plus the rounding to x's type."""
    want = ns(x.double().cpu(), steps, coef, eps)
    base = float((ns(x.float().cpu(), steps, coef, eps).double() - want).norm())
    size = float(want.norm())
    return want, 8 * base + 2.0 ** -20 * size + (HALF_STEP[x.dtype] * size if x.dtype != torch.float32 else 0.0) + 1e-30


def muon_expected(p, g, m, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, scale="spectral", **kw):
    """(p, m) after a step in float64 and the tolerances of either in the Frobenius norm."""
    p64, g64, m64 = (t.detach().cpu().double() for t in (p, g, m))
    m64 = momentum * m64 + (1 - momentum) * g64
    u = (1 - momentum) * g64 + momentum * m64 if nesterov else m64
    s, tol = 1.0, 4 * U32 * float(u.norm())
    if p64.dim() > 1:
        r, c = p64.shape[0], p64[0].numel()
        s = math.sqrt(max(1.0, r / c)) if scale == "spectral" else 0.2 * math.sqrt(max(r, c))
        # the iteration starts from the kernel's u, off by four fp32 roundings: the float32 yardstick starts from a rounded u too
        u32 = u.float()
        want, tol = ns_expected(u32.reshape(r, c), **kw)
        want = ns(u.reshape(r, c), **{**dict(steps=5), **kw})
        tol += 4 * float((ns(u32.double().reshape(r, c), **kw) - want).norm()) + 2.0 ** -20 * float(want.norm())
        u = want.reshape(p64.shape)
    new = p64 * (1 - lr * weight_decay) - lr * s * u
    return new, m64, 3 * U32 * float(p64.norm()) + lr * s * tol, 4 * U32 * float(m64.norm()) + 1e-30
