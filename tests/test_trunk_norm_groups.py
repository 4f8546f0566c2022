"""residual_norm with a gate of many small groups: its values and gradients, the workspace of its backward pass, and where it ends."""
import ctypes as C

import pytest
import torch

import trunk_ref as ref
from test_gpu_trunk import _check_norm


@pytest.fixture(scope="module", autouse=True)
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    return torch.ops.veex


def _lanes(cols):
    """Rows that a block of the backward kernel works on at a time."""
    return next((rows for width, rows in ((64, 32), (128, 16), (256, 8), (512, 4), (1024, 2)) if cols <= width), 1)


@pytest.mark.parametrize("rows", [131072, 1 << 20, 7 * 9 * 5 * 64, 6])
@pytest.mark.parametrize("cols", [1, 16, 64, 100, 128, 256, 512, 1000, 1024, 2048, 4096, 16384])
def test_workspace_does_not_grow_with_the_groups(rows, cols):
    """At most (row lanes + 1) partial rows for each block that the chip holds, of five sums, whatever the groups."""
    from vae_eeg_xai_amd import _lib
    blocks = 256 if cols > 2048 else 512
    for groups in [g for g in range(1, 2049) if rows % g == 0] + [rows // t for t in range(1, 65) if rows % t == 0]:
        floats = _lib.lib.veex_residual_norm_bwd_workspace_floats(rows, cols, groups)
        assert 0 < floats <= 5 * (_lanes(cols) + 1) * blocks * cols, groups
    assert _lib.lib.veex_residual_norm_bwd_workspace_floats(131072, 1024, 65536) * 4 < 16 << 20        # 1.3 GB with a partial row a group


def test_a_training_forward_refuses_what_the_backward_would(ops):
    from vae_eeg_xai_amd import _lib
    q = _lib.ResidualNormDesc()
    q.struct_size = C.sizeof(q)
    q.rows, q.cols, q.groups, q.eps = 1 << 23, 8, 1 << 22, 1e-3
    q.x = q.h = q.gate = q.x_out = q.u = q.stats = 1 << 20        # never dereferenced
    assert _lib.lib.veex_residual_norm_fwd(C.byref(q), None) == -1 and "groups" in _lib.lib.veex_last_error().decode()
    x, gate = torch.zeros(1 << 23, 1), torch.zeros(1 << 22, 1)
    for k in range(3):
        t = [x, x, gate]
        t[k] = t[k].clone().requires_grad_()
        with pytest.raises(ValueError, match="groups"):
            ops.residual_norm(*t)


# widths that take 8 lanes to 16 waves a row, whole and odd; a last run that is not full; row lanes without a group
MANY = [(32832, 64, 16416), (33024, 33, 16512), (16512, 128, 8256), (16386, 101, 8193), (8250, 256, 4125), (4200, 512, 2100), (2100, 1024, 1050), (2106, 1001, 1053),
        (6300, 1024, 1050), (3090, 2048, 1030), (3081, 1999, 1027), (2056, 4096, 514), (1030, 4097, 515), (1030, 8192, 515), (1026, 8191, 513), (1030, 9000, 515), (1026, 9001, 513)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,kind", [("f32", "layer"), ("bf16", "rms"), ("f16", "layer")])
@pytest.mark.parametrize("m,n,groups", MANY)
def test_many_small_groups(ops, monkeypatch, m, n, groups, dt, kind):
    """The bounds of norm_bounds with 192 roundings for its 128: a column sum here runs over up to 12 rows of a row lane, 32 row lanes, 35
    chunks of a lane of the second pass and its 16 lanes, under 90 in a row, beside the some 80 of the statistics and the formula."""
    monkeypatch.setattr(ref, "NORM_COUNT", 192)
    _check_norm(ops, m, n, groups, dt, kind, True, True)


@pytest.mark.gpu
def test_many_small_groups_without_scale_or_affine(ops, monkeypatch):
    monkeypatch.setattr(ref, "NORM_COUNT", 192)
    _check_norm(ops, 2100, 1024, 1050, "f32", "layer", True, False)
    _check_norm(ops, 2100, 1024, 1050, "bf16", "rms", True, True, parts=(False, True))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,groups", [(2100, 1024, 1050), (16386, 101, 8193), (2056, 4096, 514)])
def test_each_gradient_of_many_groups_by_itself(ops, m, n, groups):
    """Asked for alone, a gradient has the bits it has among all; the same call gives the same bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = [r(m, n), r(m, n), r(groups, n), *(r(n) for _ in range(5))]
    _, _, stats = ops.residual_norm_fwd(*t, groups, 0, 1e-3, True)
    dO, dU = r(m, n), r(m, n)
    whole = ops.residual_norm_bwd(*t, groups, 0, 1e-3, stats, dO, dU, [True] * 8)
    again = ops.residual_norm_bwd(*t, groups, 0, 1e-3, stats, dO, dU, [True] * 8)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    for k in range(8):
        one = ops.residual_norm_bwd(*t, groups, 0, 1e-3, stats, dO, dU, [i == k for i in range(8)])
        assert torch.equal(one[k], whole[k]), k
        assert all(o.numel() == 0 for i, o in enumerate(one) if i != k)


@pytest.mark.gpu
def test_a_batch_entrys_gate_for_two_tokens(ops):
    """(B, T, N) with T = 2 against the same call on a gate of x's shape: dgate sums over the two, all else is the same formula."""
    B, T, N = 3000, 2, 72
    g = torch.Generator(device="cuda").manual_seed(4)
    x, h, dO, dU = (torch.randn(B, T, N, device="cuda", generator=g) for _ in range(4))
    gate, scale = torch.randn(B, N, device="cuda", generator=g), torch.randn(N, device="cuda", generator=g)
    res = []
    for form in (gate, gate.view(B, 1, N).expand(B, T, N).contiguous()):
        leaves = [v.clone().requires_grad_() for v in (x, h, form, scale)]
        out = ops.residual_norm(*leaves, kind="rms")
        res.append([*out, *torch.autograd.grad(out, leaves, (dO, dU))])
    few, full = res
    full[4] = full[4].sum(1)
    for k, (a, b) in enumerate(zip(few, full)):
        # (the first four: the same arithmetic in another kernel; dgate: two terms; dscale: 6 000 terms in another order)
        terms = 6000 if k == 5 else 8
        a, b = a.detach(), b.detach()
        assert float((a - b).abs().max()) <= 4 * terms ** 0.5 * ref.U * 8 * float(b.abs().max()), k


@pytest.mark.gpu
def test_low_level_ops_refuse_a_gate_that_does_not_fit(ops):
    """A gate without rows beside an x with some is an error, not a missing gate; so are no groups."""
    x, none = torch.zeros(4, 8, device="cuda"), torch.zeros(0, 8, device="cuda")
    stats = torch.zeros(4, 4, device="cuda")
    rest = [None] * 5
    for gate, groups in ((none, 1), (none, 4), (None, 0), (x, 0), (x[:3], 3), (x[:2], 4)):
        with pytest.raises(ValueError):
            ops.residual_norm_fwd(x, x, gate, *rest, groups, 0, 1e-3, False)
        with pytest.raises(ValueError):
            ops.residual_norm_bwd(x, x, gate, *rest, groups, 0, 1e-3, stats, x, x, [True] * 8)
    out, u, _ = ops.residual_norm_fwd(none, none, none, *rest, 1, 0, 1e-3, True)        # no rows at all: nothing to do
    assert out.shape == (0, 8) and u.shape == (0, 8)


@pytest.mark.gpu
def test_many_groups_captured_and_on_another_stream(ops):
    """A backward pass of many groups keeps nothing between calls: captured, it is replayed on new inputs between eager calls, and gives their bits."""
    m, n, groups = 16386, 101, 8193
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = [r(m, n), r(m, n), r(groups, n), *(r(n) for _ in range(5))]
    dO, dU = r(m, n), r(m, n)

    def step():
        stats = ops.residual_norm_fwd(*t, groups, 0, 1e-3, True)[2]
        return ops.residual_norm_bwd(*t, groups, 0, 1e-3, stats, dO, dU, [True] * 8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(warm, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        t[0].copy_(r(m, n))
        t[2].copy_(r(groups, n))
        eager = [v.clone() for v in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
