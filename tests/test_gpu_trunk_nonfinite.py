"""GPU: infinities and NaN through the fp32 Dense products that run on split operands, forward and both gradients: the values fp32 gives,
in the rows and columns that hold them, and the bits of the finite call everywhere else."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module", autouse=True)
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    return torch.ops.veex


# rows and columns of whole tiles and ragged ones (packed rows padded); the last three: larger tiles, reductions split over blocks
SIZES = [(1024, 1200, 1280), (1021, 1203, 1277), (2077, 770, 1001), (4096, 1030, 2050), (200, 9000, 1000)]


def _products(ops, x, w, dy):
    """What x w, dy w^T and x^T dy give: (rows of the first operand, columns of the second)."""
    dx, dw, _ = ops.dense_bwd(dy, x, w, None, 0, 0.0, 0, 0, None, True, True, False)
    return {"y": ops.dense(x, w), "dx": dx, "dw": dw}


def _operands(x, w, dy):
    """Each product as a plain pair (A, B) with A B the product."""
    return {"y": (x, w), "dx": (dy, w.t()), "dw": (x.t(), dy)}


@pytest.mark.parametrize("m,k,n", SIZES)
def test_infinities_and_nan_in_each_operand(ops, m, k, n):
    g = torch.Generator(device="cuda").manual_seed(m)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    clean = {"x": r(m, k), "w": r(k, n) * k ** -0.5, "dy": r(m, n)}
    base = _products(ops, **clean)
    marks = {"x": (m, k), "w": (k, n), "dy": (m, n)}
    for name, (p, q) in marks.items():
        t = clean[name].clone()
        # one infinity of each sign, two that cancel in a row, a NaN beside an infinity's row, one at the end
        t[5, 7], t[9, q - 1], t[33, 1], t[33, 2], t[10, 3], t[p - 1, 0] = INF, -INF, INF, INF, NAN, INF
        dirty = dict(clean, **{name: t})
        got = _products(ops, **dirty)
        for what, (a, b) in _operands(**dirty).items():
            rows, cols = (~torch.isfinite(a)).any(1), (~torch.isfinite(b)).any(0)
            touched = rows[:, None] | cols[None, :]
            assert torch.equal(got[what][~touched], base[what][~touched]), (name, what)
            want = a.double() @ b.double()
            hit, ref = got[what][touched].double(), want[touched]
            assert torch.equal(torch.isnan(hit), torch.isnan(ref)), (name, what)
            assert torch.equal(hit[torch.isinf(ref)], ref[torch.isinf(ref)]), (name, what)
            assert not bool(torch.isfinite(ref).any()) and not bool(torch.isfinite(hit).any()), (name, what)


@pytest.mark.parametrize("m,k,n", SIZES[:3])
def test_all_nan_and_all_infinite(ops, m, k, n):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randn(*s, device="cuda", generator=g) for s in ((m, k), (k, n), (m, n)))
    for bad in (dict(x=torch.full_like(x, NAN)), dict(w=torch.full_like(w, NAN)), dict(dy=torch.full_like(dy, NAN))):
        args = dict(x=x, w=w, dy=dy) | bad
        got = _products(ops, **args)
        for what, (a, b) in _operands(**args).items():
            assert bool((torch.isnan(got[what]) == (torch.isnan(a).any() | torch.isnan(b).any())).all()), what
    pos = torch.full_like(x, INF)
    y = ops.dense(pos, w.abs() + 1)
    assert bool((y == INF).all())
