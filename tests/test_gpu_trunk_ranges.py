"""GPU: torch.ops.veex.dense near the ends of its types' ranges, against the 64-bit forms of trunk_ref.py."""
import pytest
import torch

import trunk_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    return torch.ops.veex


# general product; the same with odd sizes; aligned and packed tiles, whose reductions are split for dw, or for dx
SIZES = [(96, 64, 72), (41, 333, 77), (300, 264, 520), (1303, 1001, 207), (2048, 264, 136), (264, 136, 2048)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("act,rate,size", [(None, 0.5, 60000.0), ("relu", 0.9, 65504.0), ("gelu", 0.0, 65504.0), ("gelu", 0.5, 65504.0), ("silu", 0.99, 65504.0), ("sigmoid", 0.5, 65504.0),
                                           (None, 0.5, 2.0 ** -20), ("gelu", 0.0, 2.0 ** -18), ("silu", 0.25, 2.0 ** -20)])
def test_fp16_gradients_of_large_and_small_dy(ops, m, k, n, act, rate, size):
    """dy up to the type's largest number, so that dz = D'(dy) act'(z) is past it while dx and dw are not; and dy of the type's last few
    steps.  dz is held in fp16 times c = (1 - rate) 7/8 (no 7/8 where the slope is at most 1): one rounding, of which half a step of
    the smallest numbers is t / c of dz, and three fp32 factors; the rest is dense_bounds."""
    t16 = torch.float16
    g = torch.Generator().manual_seed(m + 3 * n)
    # weights and inputs small enough that sums over all of dy stay inside the type: scale^2 times the terms' count is about 1
    large = size > 1.0
    scale = 1.0 - round(rate * 65536) / 65536
    down = 0.1 * scale ** 0.5 if large else 1.0
    w = (torch.randn(k, n, generator=g) * down * n ** -0.5).to(t16)
    x = (torch.randn(m, k, generator=g) * down * m ** -0.5).to(t16)
    b = torch.randn(n, generator=g).to(t16)
    b = torch.where(b.abs() < 0.25, torch.tensor(0.5, dtype=t16), b)                 # (no relu near its kink: |x w| is below 0.1)
    dy = ((torch.rand(m, n, generator=g) * 2 - 1) * size).to(t16)
    dy[::3, ::5] = size
    dy[1::3, ::7] = -size
    X, W, B, DY = (v.double() for v in (x, w, b, dy))
    assert float((X @ W).abs().max()) < 0.2 or act != "relu"
    f = ref.keep_factor(m, n, rate, 9, 4) if rate else None
    leaves = [v.requires_grad_() for v in (X, W, B)]
    want = torch.autograd.grad(ref.dense(X, W, B, act, None, f), leaves, DY)
    X, W, B = (v.detach() for v in (X, W, B))
    if large:
        assert all(float(v.abs().max()) < 65504 for v in want[:2]), "the case's own gradients have to be finite"
    _, ex, ew, _ = ref.dense_bounds(t16, X, W, B, act, None, f, DY)
    z = (X @ W + B).requires_grad_()
    slope = torch.autograd.grad(ref.ACT[act](z).sum(), z)[0] if act is not None else torch.ones_like(z)
    dz = DY * (1.0 if f is None else f) * slope
    e = ref.tiny(t16) / (scale * 0.875) + 4 * ref.U * dz.abs()
    ex, ew = ex + 1.01 * (e @ W.t().abs()), ew + 1.01 * (X.t().abs() @ e)
    dev = [v.cuda().requires_grad_() for v in (x, w, b)]
    y = ops.dense(*dev, act, None, rate, 9, 4)
    got = torch.autograd.grad(y, dev[:2], dy.cuda())
    ref.within(got[0], want[0], ex, "dx")
    ref.within(got[1], want[1], ew, "dw")


@pytest.mark.parametrize("m,k,n", [(16, 64, 16), (40, 33, 21), (300, 264, 520)])
@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
def test_bf16_sums_between_its_range_and_fp32s(ops, m, k, n, act):
    """A z that fp32 holds and bf16 rounds to an infinity: the gradient is the activation's limit, not NaN, as for fp16."""
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with torch.no_grad():
        x[:, 0], x[:, 1] = 255 * 2.0 ** 120, 2.0 ** 119
    w = torch.zeros(k, n, dtype=torch.bfloat16, device="cuda")
    w[:2, ::2], w[:2, 1::2] = 1.0, -1.0
    assert float((x.detach().float() @ w.float())[0, 0]) == 511 * 2.0 ** 119
    r = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    for residual in (None, r):
        y = ops.dense(x, w, None, act, residual)
        assert bool((y[:, ::2] == float("inf")).all()) and not y[:, 1::2].any()
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool((dx[:, :2] == (n + 1) // 2).all()) and not dx[:, 2:].any()
