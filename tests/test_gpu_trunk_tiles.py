"""Every matrix-core tile of torch.ops.veex.dense, for each product and with its reduction whole and split, on random data with reductions of many
stages and ragged edges, against the 64-bit forms (evaluated on the GPU in float64; the bounds are trunk_ref.py's)."""
import ctypes as C

import pytest
import torch

import trunk_ref as ref

PRODUCTS = ("y", "dx", "dw")
TILES = {3: "256x256", 4: "256x128", 5: "128x128"}
# rows, k, n: chosen so that the plans below reach all of them; odd sizes are packed, the others lie as they are (16-bit types)
CASES = {
    "f32": [(1263, 1201, 1055), (1421, 1283, 1459), (9152, 392, 448), (392, 6368, 6440), (5272, 2752, 304)],
    "bf16": [(1981, 363, 2225), (401, 3901, 1023), (17896, 296, 648), (288, 688, 17424), (651, 17667, 331), (15512, 408, 2056), (392, 8520, 4104), (1544, 528, 16968)],
}
CASES["f16"] = CASES["bf16"]


def _plans(dt, m, k, n):
    """(tile, whether its reduction is split, reduction length of a block) of each product."""
    from vae_eeg_xai_amd import _lib
    d = _lib.DenseDesc()
    d.struct_size = C.sizeof(d)
    d.rows, d.k, d.n, d.ldx, d.dtype = m, k, n, k, ("f32", "bf16", "f16").index(dt)
    plans = [_lib.lib.veex_dense_plan(C.byref(d), q) for q in range(3)]
    assert min(plans) >= 0
    return [(TILES.get(p & 255), p >> 8 > 1, length / (p >> 8)) for p, length in zip(plans, (k, n, m))]


@pytest.mark.parametrize("dt", CASES)
def test_the_cases_reach_every_tile(dt):
    """A change of the rules that leaves a kernel without a case fails here.  256 k's or more a block: every stage of the ring is used again."""
    reached = {(q, tile, split) for c in CASES[dt] for q, (tile, split, length) in zip(PRODUCTS, _plans(dt, *c)) if length >= 256}
    tiles = ("256x128", "128x128") if dt == "f32" else TILES.values()
    assert reached >= {(q, t, s) for q in PRODUCTS for t in tiles for s in (False, True)}


def test_plans_of_other_paths_and_refusals():
    from vae_eeg_xai_amd import _lib
    d = _lib.DenseDesc()
    d.struct_size = C.sizeof(d)
    for (m, k, n, dt), path in (((1, 1024, 1024, 1), 2), ((1, 4096, 4096, 1), 1), ((5, 6400, 100, 0), 1), ((512, 6400, 100, 0), 0), ((64, 64, 64, 1), 5)):
        d.rows, d.k, d.n, d.ldx, d.dtype = m, k, n, k, dt
        assert _lib.lib.veex_dense_plan(C.byref(d), 0) & 255 == path, (m, k, n, dt)
    assert _lib.lib.veex_dense_plan(C.byref(d), 3) == -1 and _lib.lib.veex_dense_plan(C.byref(d), -1) == -1
    d.rows = 0
    assert _lib.lib.veex_dense_plan(C.byref(d), 0) == -1
    d.rows, d.k = 4, 0
    assert _lib.lib.veex_dense_plan(C.byref(d), 0) == -1


def _within(got, want, bound, what):
    excess = (got.double() - want).abs() / bound
    assert bool(torch.isfinite(excess).all()), f"{what}: not finite"
    at = int(excess.argmax())
    assert float(excess.max()) <= 1.0, f"{what}: {float(excess.max()):.2f} times the bound at {divmod(at, got.shape[-1])}"


@pytest.mark.gpu
@pytest.mark.parametrize("dt,m,k,n", [(dt, *c) for dt, cases in CASES.items() for c in cases])
def test_large_products(dt, m, k, n):
    import vae_eeg_xai_amd.ops  # noqa: F401
    ops, dtype, rate = torch.ops.veex, ref.TYPES[dt], 0.25
    g = torch.Generator(device="cuda").manual_seed(m + n)
    r = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)  # noqa: E731
    leaves = [r(m, k).requires_grad_(), r(k, n, scale=k ** -0.5).requires_grad_(), r(n, scale=0.5).requires_grad_()]
    res, dy = r(m, n), r(m, n)
    y = ops.dense(*leaves, "silu", res, rate, 7, 5)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    f = (ops.dropout(torch.ones(m, n, device="cuda"), rate, 7, 5) != 0).double() / (1 - rate)       # (1/4 is a whole number of 1/65536)
    X, W, B = (t.detach().double() for t in leaves)
    bounds = ref.dense_bounds(dtype, X, W, B, "silu", res.double(), f, dy.double())
    exact = [t.requires_grad_() for t in (X, W, B)]
    Y = ref.dense(*exact, "silu", res.double(), f)
    want = [Y.detach(), *torch.autograd.grad(Y, exact, dy.double())]
    for what, a, b, e in zip(("y", "dx", "dw", "db"), got, want, bounds):
        _within(a, b, e, what)
