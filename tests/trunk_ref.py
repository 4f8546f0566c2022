"""Plain 64-bit restatements of the dense-trunk operators (dense, dropout, residual_norm) for their tests, and the error
bounds the tests hold the kernels to.  No code of the package is used.

Rounding units: h(T) = eps(T) / 2 is the largest relative error of one rounding to T; U = 2^-24 that of fp32.  A sum of n fp32
terms in any order is off by at most about LAM sqrt(n) U times the sum of the terms' magnitudes, but for a probability of
2 exp(-LAM^2 / 2) per value (rounding errors as independent, mean-zero variables: Higham & Mary, "A new approach to
probabilistic rounding error analysis", 2019); LAM = 8 makes that 3e-14."""
import math

import numpy as np
import torch

U = 2.0 ** -24
LAM = 8.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the smallest numbers (fp16 loses relative precision below 2^-14)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def philox(counter, key):
    """Philox-4x32-10 on arrays of uint32 words (4 x N) under the key's two words."""
    c = [np.asarray(a, dtype=np.uint64) for a in counter]
    k0, k1 = int(key[0]), int(key[1])
    m32 = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m32, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return [a.astype(np.uint32) for a in c]


def keep_factor(rows, cols, rate, seed, first_row=0):
    """(rows, cols) float64: 0 where an element is dropped, 1 / (1 - rate) (rate to 1/65536) where it stays."""
    cut = round(rate * 65536)
    blocks = (cols + 7) // 8
    r = [(first_row + i) % 2 ** 64 for i in range(rows)]
    lo = np.array([v & 0xFFFFFFFF for v in r], dtype=np.uint64)[:, None]
    hi = np.array([v >> 32 for v in r], dtype=np.uint64)[:, None]
    z = np.zeros((rows, blocks), dtype=np.uint64)
    w = philox([z + np.arange(blocks, dtype=np.uint64), z + np.uint64(0x44524F50), z + lo, z + hi], (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    u = np.zeros((rows, blocks, 8), dtype=np.int64)
    for e in range(8):
        u[:, :, e] = (w[e >> 1] >> np.uint32(16 * (e & 1))) & np.uint32(0xFFFF)
    return torch.from_numpy((u.reshape(rows, -1)[:, :cols] >= cut) * (65536.0 / (65536 - cut)))


ACT = {None: lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid}
# largest slope and largest curvature of each
SLOPE = {None: 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1, "sigmoid": 0.25}
CURVE = {None: 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5, "sigmoid": 0.1}


def dense(x, w, b=None, act=None, residual=None, factor=None):
    z = x @ w if b is None else x @ w + b
    y = ACT[act](z)
    y = y if factor is None else y * factor
    return y if residual is None else y + residual


def dense_bounds(dtype, x, w, b, act, residual, factor, dy):
    """Largest differences of y, dx, dw, db (elementwise, float64 tensors) that the roundings allow; x, w, ... in float64,
    already the rounded values.  z's sum runs in fp32 over exact products of 16-bit types; an fp32 product may be made of
    bf16 terms, off by 2^-25 and six times as many summands.  What is rounded to the type: y, the stored z, dz, and the results."""
    h, t = half(dtype), tiny(dtype)
    n6 = 6 if dtype == torch.float32 else 1
    m, k = x.shape

    def mm(a, c, n):       # error of a product whose operands are exact
        return (LAM * math.sqrt(n6 * n) * U + 2.0 ** -25) * (a.abs() @ c.abs())

    z = x @ w + (0.0 if b is None else b)
    ez = mm(x, w, k) + 2 * U * z.abs()
    f = torch.ones_like(z) if factor is None else factor
    y = dense(x, w, b, act, residual, factor)
    ey = f * (SLOPE[act] * ez + 8 * U * (1 + z.abs())) + 2 * U * y.abs()
    ey = ey + h * (y.abs() + ey) + t
    if dy is None:
        return ey, None, None, None
    zr = z.clone().requires_grad_()
    d1 = torch.autograd.grad(ACT[act](zr).sum(), zr)[0] if act is not None else torch.ones_like(z)
    g = dy * f
    dz = g * d1
    # slope at the stored z; evaluating it costs some U of 1 + |z|; nothing is evaluated or rounded without an activation
    ed = torch.zeros_like(z) if act is None else g.abs() * (CURVE[act] * (h * z.abs() + t + ez) + 8 * U * (1 + z.abs()))
    if factor is not None:
        ed = ed + 2 * U * dz.abs()
    er = ed if act is None and factor is None else ed + h * (dz.abs() + ed) + t        # dz as the products read it
    dx, dw, db = dz @ w.t(), x.t() @ dz, dz.sum(0)
    ex = er @ w.t().abs() + mm(dz.abs() + er, w.t(), w.shape[1])
    ew = x.t().abs() @ er + mm(x.t(), dz.abs() + er, m)
    eb = ed.sum(0) + LAM * math.sqrt(m) * U * (dz.abs() + ed).sum(0)
    return ey, *(e + h * (r.abs() + e) + t for e, r in ((ex, dx), (ew, dw), (eb, db)))


def norm(v, w, b, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    v = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def residual_norm(x, h, gate, scale, post_w, post_b, pre_w, pre_b, kind, eps):
    """x, h (rows, cols); gate (groups, cols)."""
    out = x
    if h is not None:
        n = norm(h, post_w, post_b, kind, eps)
        n = n if scale is None else n * scale
        out = x + (n if gate is None else n * gate.repeat_interleave(x.shape[0] // gate.shape[0], 0))
    return out, norm(out, pre_w, pre_b, kind, eps)


NORM_COUNT = 128     # roundings that may meet in one value: a statistic is a sum of at most 16 values a lane, 6 to 10 tree
#                      levels and a square root (under 32 U, two of them, on values that themselves carry 32 U), ten elementwise
#                      steps, and the rows of a chunk and chunks of a column sum in the tests' sizes (under 40)


def norm_bounds(dtype, x, h, gate, scale, post_w, post_b, pre_w, pre_b, kind, eps, dx_out, du):
    """Largest differences of (x_out, u) and of the eight gradients: each formula evaluated on magnitudes (every difference as a
    sum, every centred value as |v| + mean|v|), times NORM_COUNT U, plus the rounding of the result."""
    h_, t = half(dtype), tiny(dtype)
    a = lambda v, other=1.0: other if v is None else v.abs()  # noqa: E731
    layer = kind == "layer"

    def hat(v):
        mean = v.mean(-1, keepdim=True) if layer else 0.0
        r = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
        return (v.abs() + (v.abs().mean(-1, keepdim=True) if layer else 0.0)) * r, r

    res = {}
    rows = x.shape[0]
    full = 1.0 if gate is None else gate.abs().repeat_interleave(rows // gate.shape[0], 0)
    out_abs = x.abs()
    if h is not None:
        xh, r1 = hat(h)
        n = xh * a(post_w) + a(post_b, 0.0)
        out_abs = out_abs + a(scale) * full * n
        res["x_out"] = out_abs
    out = residual_norm(x, h, gate, scale, post_w, post_b, pre_w, pre_b, kind, eps)[0]
    _, r2 = hat(out)
    rh = (out_abs + (out_abs.mean(-1, keepdim=True) if layer else 0.0)) * r2
    res["u"] = rh * a(pre_w) + a(pre_b, 0.0)
    if du is not None:
        tt = du.abs() * a(pre_w)
        D = dx_out.abs() + r2 * (tt + rh * (tt * rh).mean(-1, keepdim=True) + (tt.mean(-1, keepdim=True) if layer else 0.0))
        res["x"], res["pre_w"], res["pre_b"] = D, (du.abs() * rh).sum(0), du.abs().sum(0)
        if h is not None:
            dn = D * a(scale) * full
            e = dn * a(post_w)
            res["h"] = r1 * (e + xh * (e * xh).mean(-1, keepdim=True) + (e.mean(-1, keepdim=True) if layer else 0.0))
            res["post_w"], res["post_b"] = (dn * xh).sum(0), dn.sum(0)
            res["scale"] = (D * n * full).sum(0)
            if gate is not None:
                res["gate"] = (D * n * a(scale)).reshape(gate.shape[0], -1, x.shape[1]).sum(1)
    return {k: (lambda ref, e=NORM_COUNT * U * v: e + h_ * (ref.abs() + e) + t) for k, v in res.items()}


def within(got, ref, bound, what=""):
    """Elementwise |got - ref| <= bound, with the worst place in the message."""
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if got.numel() == 0:
        return
    excess = ((got - ref).abs() / bound)
    assert bool(torch.isfinite(excess).all()), f"{what}: not finite"
    at = int(excess.argmax())
    assert float(excess.max()) <= 1.0, f"{what}: {float(excess.max()):.2f} times the bound at {at}: {float(got.reshape(-1)[at])} for {float(ref.reshape(-1)[at])}"
