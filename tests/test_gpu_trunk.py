"""GPU: torch.ops.veex.dense / dropout / residual_norm against their plain 64-bit restatements (trunk_ref.py) at the sizes, types,
strides and values where they can go wrong, within bounds derived there; gradients also against differences; then used together,
on other streams, captured and replayed."""
import math

import pytest
import torch

import trunk_ref as ref

pytestmark = pytest.mark.gpu
TYPES = ref.TYPES


@pytest.fixture(scope="module", autouse=True)
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    return torch.ops.veex


def _rand(g, *shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def _case(seed, m, k, n, dtype, residual, act):
    g = torch.Generator().manual_seed(seed)
    x, w = _rand(g, m, k, dtype=dtype), _rand(g, k, n, dtype=dtype, scale=k ** -0.5)
    b, dy = _rand(g, n, dtype=dtype, scale=0.5), _rand(g, m, n, dtype=dtype)
    r = _rand(g, m, n, dtype=dtype) if residual else None
    if act == "relu":     # no sum near the kink, where the rounding of a sum decides an element: move those rows' bias away
        z = x.double() @ w.double() + b.double()
        for _ in range(200):
            near = (z.abs() < 1e-3).any(0)
            if not near.any():
                break
            b = torch.where(near, b + torch.tensor(0.013, dtype=dtype), b)
            z = x.double() @ w.double() + b.double()
    return x, w, b, dy, r


def _check_dense(ops, m, k, n, dt, act, residual, rate, train, first_row=0):
    dtype = TYPES[dt]
    x, w, b, dy, r = _case(m * 7 + k * 3 + n, m, k, n, dtype, residual, act)
    xd, wd, bd = (t.cuda().requires_grad_(train) for t in (x, w, b))
    rd = None if r is None else r.cuda().requires_grad_(train)
    y = ops.dense(xd, wd, bd, act, rd, rate, 1234, first_row)
    X, W, B, DY = (t.double() for t in (x, w, b, dy))
    R = None if r is None else r.double()
    f = ref.keep_factor(m, n, rate, 1234, first_row) if rate else None
    leaves = [t.requires_grad_() for t in (X, W, B)]
    Y = ref.dense(X, W, B, act, R, f)
    gr = torch.autograd.grad(Y, leaves, DY) if train else (None,) * 3
    ey, ex, ew, eb = ref.dense_bounds(dtype, X.detach(), W.detach(), B.detach(), act, R, f, DY if train else None)
    if act == "relu":
        z = (X @ W + B).detach().abs()
        assert float(z.min()) > 1e-4, "the inputs of this case leave a sum at the kink"
    ref.within(y, Y.detach(), ey, "y")
    if not train:
        return
    got = torch.autograd.grad(y, [xd, wd, bd] + ([rd] if residual else []), dy.cuda())
    for what, a, c, e in zip(("dx", "dw", "db"), got, gr, (ex, ew, eb)):
        ref.within(a, c, e, what)
    if residual:
        assert torch.equal(got[3].cpu(), dy)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (2, 7, 3), (1, 6400, 100), (3, 28, 4096), (63, 33, 65), (64, 64, 64), (65, 100, 56),
                                   (129, 32, 8), (70, 12, 20), (200, 36, 100), (130, 257, 333), (257, 1001, 127), (512, 96, 320), (520, 264, 264)])
def test_dense_sizes(ops, m, k, n, dt):
    _check_dense(ops, m, k, n, dt, "gelu", True, 0.0, True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k,n", [(300, 1000, 520), (1030, 264, 1001), (129, 4104, 260), (260, 5000, 136), (8000, 2000, 60), (1500, 72, 2056), (2051, 513, 259), (1500, 1032, 1104), (1303, 1001, 1207)])
def test_dense_large(ops, m, k, n, dt):
    """On the 16-bit matrix cores: tiles that end inside the tensors, odd sizes that are packed, split reductions."""
    _check_dense(ops, m, k, n, dt, "silu", True, 0.1, True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k,n", [(1, 65536, 1), (1, 257, 1000), (1, 700, 100), (2, 700, 264), (3, 1001, 77), (5, 640, 4096), (8, 4096, 136), (2, 640, 4096), (1, 4096, 136), (7, 700, 264), (1, 1024, 1000), (2, 100, 6400), (4, 1023, 68), (8, 64, 1032), (1, 7, 9368), (3, 1025, 200)])
def test_dense_few_rows(ops, m, k, n, dt):
    _check_dense(ops, m, k, n, dt, "gelu", True, 0.2, False)
    _check_dense(ops, m, k, n, dt, "sigmoid", False, 0.0, True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("residual,rate", [(False, 0.0), (True, 0.0), (False, 0.25), (True, 0.5)])
def test_dense_epilogues(ops, dt, act, residual, rate):
    _check_dense(ops, 37, 40, 72, dt, act, residual, rate, True, first_row=(1 << 33) + 5)


def test_dense_without_bias_and_with_some_gradients(ops):
    g = torch.Generator().manual_seed(5)
    x, w, dy = (_rand(g, *s, dtype=torch.float32).cuda() for s in ((33, 40), (40, 24), (33, 24)))
    for needs in ((True, False), (False, True)):
        xs, ws = x.clone().requires_grad_(needs[0]), w.clone().requires_grad_(needs[1])
        y = ops.dense(xs, ws, None, "silu")
        got = torch.autograd.grad(y, [t for t in (xs, ws) if t.requires_grad], dy)
        X, W = x.double().cpu().requires_grad_(), w.double().cpu().requires_grad_()
        gr = torch.autograd.grad(ref.dense(X, W, None, "silu"), (X, W), dy.double().cpu())
        e = ref.dense_bounds(torch.float32, X.detach(), W.detach(), None, "silu", None, None, dy.double().cpu())
        ref.within(got[0], gr[0 if needs[0] else 1], e[1 if needs[0] else 2])
    r = torch.zeros(33, 24, device="cuda", requires_grad=True)       # only the residual learns
    dr, = torch.autograd.grad(ops.dense(x, w, None, "silu", r), r, dy)
    assert torch.equal(dr, dy)
    with pytest.raises(RuntimeError):                                 # differentiable once
        xs = x.clone().requires_grad_()
        d, = torch.autograd.grad(ops.dense(xs, w, None, "silu"), xs, dy, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_dense_strides_alignment_and_shapes(ops, dt):
    """Leading indices, a row stride, transposed and misaligned tensors, an expanded dy: the bits of contiguous copies."""
    dtype = TYPES[dt]
    g = torch.Generator().manual_seed(9)
    wide = _rand(g, 48, 200, dtype=dtype).cuda()
    w = _rand(g, 64, 40, dtype=dtype, scale=0.1).cuda()
    b = _rand(g, 40, dtype=dtype).cuda()
    base = ops.dense(wide[:, 8:72].contiguous(), w, b, "gelu")
    assert torch.equal(ops.dense(wide[:, 8:72], w, b, "gelu"), base)                       # row stride 200, 16-byte aligned
    e = 2 * ref.dense_bounds(dtype, wide[:, 9:73].double().cpu(), w.double().cpu(), b.double().cpu(), "gelu", None, None, None)[0]
    ref.within(ops.dense(wide[:, 9:73], w, b, "gelu"), ops.dense(wide[:, 9:73].contiguous(), w, b, "gelu").double().cpu(), e)      # another kernel may serve it
    xt = wide[:, :64].t().contiguous().t()
    assert torch.equal(ops.dense(xt, w, b, "gelu"), ops.dense(wide[:, :64].contiguous(), w, b, "gelu"))
    wt = w.t().contiguous().t()
    assert torch.equal(ops.dense(wide[:, 8:72], wt, b, "gelu"), base)
    assert torch.equal(ops.dense(wide[:, 8:72].contiguous().view(2, 4, 6, 64), w, b, "gelu"), base.view(2, 4, 6, 40))
    assert torch.equal(ops.dense(wide[5, 8:72], w, b, "gelu"), ops.dense(wide[5:6, 8:72], w, b, "gelu")[0])
    one = wide[0, 8:72].expand(7, 64)
    assert torch.equal(ops.dense(one, w, b, "gelu"), ops.dense(one.contiguous(), w, b, "gelu"))
    buf = torch.empty(64 * 40 + 1, dtype=dtype, device="cuda")[1:].view(64, 40)            # weights off a 16-byte border
    buf.copy_(w)
    e = 2 * ref.dense_bounds(dtype, wide[:, 8:72].double().cpu(), w.double().cpu(), b.double().cpu(), "gelu", None, None, None)[0]
    ref.within(ops.dense(wide[:, 8:72], buf, b, "gelu"), base.double().cpu(), e)
    x = wide[:, 8:72].contiguous().requires_grad_()
    y = ops.dense(x, w, b, "gelu")
    d1, = torch.autograd.grad(y, x, torch.ones(1, 1, dtype=dtype, device="cuda").expand(48, 40), retain_graph=True)
    d2, = torch.autograd.grad(y, x, torch.ones(48, 40, dtype=dtype, device="cuda"))
    assert torch.equal(d1, d2)


def test_dense_fp16_sums_beyond_its_range(ops):
    """z past 65504: y is an infinity (or 0 on the other side), and the gradient is the activation's limit, not NaN."""
    x = torch.full((16, 64), 100.0, dtype=torch.float16, device="cuda")
    w = torch.full((64, 16), 20.0, dtype=torch.float16, device="cuda")
    w[:, 8:] = -20.0
    for act in ("gelu", "silu", "relu"):
        xs = x.clone().requires_grad_()
        y = ops.dense(xs, w, None, act)
        assert bool(torch.isinf(y[:, :8]).all()) and not y[:, 8:].any()
        dx, = torch.autograd.grad(y, xs, torch.ones_like(y))
        assert torch.equal(dx, torch.full_like(dx, 160.0))


def test_low_level_ops_refuse_what_does_not_fit(ops):
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(8, 6, device="cuda")
    y = torch.zeros(4, 6, device="cuda")
    for bad in (lambda: ops.dense_fwd(x, torch.zeros(9, 6, device="cuda"), None, 0, None, 0.0, 0, 0, None, False),
                lambda: ops.dense_fwd(x, w, torch.zeros(5, device="cuda"), 0, None, 0.0, 0, 0, None, False),
                lambda: ops.dense_fwd(x, w.cpu(), None, 0, None, 0.0, 0, 0, None, False),
                lambda: ops.dense_bwd(y[:3], x, w, None, 0, 0.0, 0, 0, None, True, True, True),
                lambda: ops.dense_bwd(y, x, w, None, 1, 0.0, 0, 0, None, True, True, True),
                lambda: ops.dense_bwd(y, x, w, y[:, :5], 1, 0.0, 0, 0, None, True, True, True),
                lambda: ops.dropout_fwd(x, 0.5, 1, 0, w, None),
                lambda: ops.residual_norm_fwd(x, x[:3], None, None, None, None, None, None, 1, 0, 1e-3, False),
                lambda: ops.residual_norm_fwd(x, x, torch.zeros(3, 8, device="cuda"), None, None, None, None, None, 3, 0, 1e-3, False),
                lambda: ops.residual_norm_bwd(x, x, None, None, None, None, None, None, 1, 0, 1e-3, torch.zeros(3, 4, device="cuda"), x, x, [True] * 8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.dense_fwd(x, w, None, 9, None, 0.0, 0, 0, None, False)


def test_dense_no_rows(ops):
    x, w, b = torch.zeros(0, 16, device="cuda", requires_grad=True), torch.ones(16, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    y = ops.dense(x, w, b, "relu", None, 0.5, 1)
    assert y.shape == (0, 8)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 8, device="cuda"))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_dense_infinities_and_nan_stay_in_their_rows(ops, dt):
    """A NaN row gives a NaN row, an infinity no finite value where it weighs in; no other row changes; relu passes NaN on."""
    dtype = TYPES[dt]
    for m, k, n in ((40, 48, 56), (512, 256, 256), (1024, 1200, 1280)):        # the last: fp32 by split terms
        g = torch.Generator().manual_seed(2)
        x, w = _rand(g, m, k, dtype=dtype), _rand(g, k, n, dtype=dtype, scale=0.2)
        w[:, 3] = w[:, 3].abs() + torch.finfo(dtype).eps
        clean = ops.dense(x.cuda(), w.cuda(), None, "relu")
        x[5, 7], x[9, 2] = float("nan"), float("inf")
        got = ops.dense(x.cuda(), w.cuda(), None, "relu")
        rest = [i for i in range(m) if i not in (5, 9)]
        assert torch.equal(got[rest], clean[rest])
        assert bool(torch.isnan(got[5]).all())
        plain = torch.relu(x[9:10].double() @ w.double())[0]
        assert bool((~torch.isfinite(got[9].cpu()) | (plain == 0)).all()) and float(plain[3]) == math.inf
        assert bool((got[9].cpu().double() == plain).all())


def test_dense_gradient_against_differences(ops):
    """The device's gradients, along a random direction, against differences of the 64-bit forward."""
    m, k, n = 70, 45, 52
    x, w, b, dy, r = _case(3, m, k, n, torch.float32, True, "silu")
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r)]
    y = ops.dense(*leaves[:3], "silu", leaves[3], 0.25, 77)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    f = ref.keep_factor(m, n, 0.25, 77)
    g = torch.Generator().manual_seed(4)
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=g).double() * 1e-5
        at = lambda s: float((ref.dense(*[t.double() + (s * d if i == q else 0) for q, t in enumerate((x, w, b))], "silu",  # noqa: E731
                                        r.double() + (s * d if i == 3 else 0), f) * dy.double()).sum())
        want = (at(1) - at(-1)) / 2
        size = float((gr.double().cpu() * d).abs().sum())
        assert abs(want - float((gr.double().cpu() * d).sum())) < 1e-5 * size + 1e-9


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 8), (3, 9), (5, 100), (64, 512), (33, 1001), (700, 264)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(ops, dt, m, n, residual):
    dtype = TYPES[dt]
    g = torch.Generator().manual_seed(m + n)
    x, r, dy = (_rand(g, m, n, dtype=dtype) for _ in range(3))
    f = ref.keep_factor(m, n, 0.3, -5, first_row=11)
    xd, rd = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    y = ops.dropout(xd, 0.3, -5, 11, rd if residual else None)
    want = x.double() * f + (r.double() if residual else 0.0)
    e = 2 * ref.U * (x.double() * f).abs() + 2 * ref.U * want.abs()
    ref.within(y, want, e + ref.half(dtype) * (want.abs() + e) + ref.tiny(dtype), "y")
    assert torch.equal((ops.dropout(torch.ones_like(xd), 0.3, -5, 11) != 0).cpu(), f != 0)
    dx, *dr = torch.autograd.grad(y, [xd] + ([rd] if residual else []), dy.cuda())
    want = dy.double() * f
    ref.within(dx, want, (2 * ref.U + ref.half(dtype)) * want.abs() + ref.tiny(dtype), "dx")
    assert not residual or torch.equal(dr[0].cpu(), dy)


def test_dropout_rates_rows_and_values(ops):
    x = torch.randn(64, 200, device="cuda")
    assert torch.equal(ops.dropout(x, 0.0, 1), x)
    assert torch.equal(ops.dropout(x, 1e-6, 1), x)                           # below half of 1/65536: none
    assert int((ops.dropout(x, 65535 / 65536, 1) != 0).sum()) < 30           # one in 65536 stays
    whole = ops.dropout(x, 0.5, 9, 100)
    assert torch.equal(torch.cat([ops.dropout(x[:17], 0.5, 9, 100), ops.dropout(x[17:], 0.5, 9, 117)]), whole)
    assert torch.equal(ops.dropout(x.view(4, 16, 200), 0.5, 9, 100).view(64, 200), whole)
    xt = x.t().contiguous().t()
    assert torch.equal(ops.dropout(xt, 0.5, 9, 100), whole)
    odd = torch.empty(64 * 200 + 1, device="cuda")[1:].view(64, 200).copy_(x)  # off a 16-byte border
    assert torch.equal(ops.dropout(odd, 0.5, 9, 100), whole)
    assert not torch.equal(ops.dropout(x, 0.5, 10, 100), whole)
    far = ops.dropout(x, 0.5, 9, (1 << 32) - 3)                              # rows that cross 2^32
    assert torch.equal((far != 0).cpu(), ref.keep_factor(64, 200, 0.5, 9, (1 << 32) - 3) != 0)
    y = x.clone()
    y[3], y[5] = float("inf"), float("nan")
    f = ref.keep_factor(64, 200, 0.5, 9, 100)
    z = ops.dropout(y, 0.5, 9, 100).cpu()
    assert bool((z[3][f[3] == 0] == 0).all()) and bool(torch.isinf(z[3][f[3] != 0]).all())
    assert bool((z[5][f[5] == 0] == 0).all()) and bool(torch.isnan(z[5][f[5] != 0]).all())
    assert ops.dropout(x[:0], 0.5, 1).shape == (0, 200)
    xs = x.clone().requires_grad_()                                          # its own backward, and that one's
    d, = torch.autograd.grad(ops.dropout(xs, 0.5, 9, 100) .pow(2).sum(), xs, create_graph=True)
    dd, = torch.autograd.grad(d.sum(), xs)
    assert torch.allclose(dd.cpu().double(), 2 * f * f)


def test_dropout_counter_is_read_when_the_kernel_runs_and_kept_for_the_backward_pass(ops):
    x = torch.randn(40, 100, device="cuda", requires_grad=True)
    w = torch.randn(100, 50, device="cuda", requires_grad=True)
    c = torch.tensor([1000], dtype=torch.int64, device="cuda")
    y, z = ops.dropout(x, 0.4, 3, 5, None, c), ops.dense(x, w, None, "silu", None, 0.4, 3, 5, c)
    c.add_(40)                                                               # the next step's rows, before this step's backward
    want = ops.dropout(x, 0.4, 3, 1005), ops.dense(x, w, None, "silu", None, 0.4, 3, 1005)
    for a, b in zip((y, z), want):
        assert torch.equal(a, b)
        dy = torch.randn_like(a)
        assert torch.equal(torch.autograd.grad(a, x, dy)[0], torch.autograd.grad(b, x, dy)[0])
    assert torch.equal(ops.dropout(x, 0.4, 3, 5, None, c), ops.dropout(x, 0.4, 3, 1045))


# ------------------------------------------------------------------ residual_norm
def _check_norm(ops, m, n, groups, dt, kind, gate, affine, train=True, parts=(True, True), shape=None, scale_x=1.0):
    dtype = TYPES[dt]
    g = torch.Generator().manual_seed(m * 31 + n + groups)
    t = {"x": _rand(g, m, n, dtype=dtype, scale=scale_x), "h": _rand(g, m, n, dtype=dtype, scale=0.8, shift=0.3)}
    t["gate"] = None if not gate else _rand(g, groups, n, dtype=dtype, scale=0.4, shift=1.0)
    t["scale"] = _rand(g, n, dtype=dtype, scale=0.2, shift=0.6) if affine else None
    for p in ("post", "pre"):
        t[p + "_w"] = _rand(g, n, dtype=dtype, scale=0.2, shift=1.0) if affine else None
        t[p + "_b"] = _rand(g, n, dtype=dtype, scale=0.3) if affine and kind == "layer" else None
    dout, du = _rand(g, m, n, dtype=dtype), _rand(g, m, n, dtype=dtype)
    dev = {k: None if v is None else v.cuda().requires_grad_(train) for k, v in t.items()}
    call = [dev[k] for k in ("x", "h", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b")]
    out, u = ops.residual_norm(*call, kind, 1e-3)
    R = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    args = [R[k] for k in ("x", "h", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b")]
    OUT, UU = ref.residual_norm(*args, kind, 1e-3)
    D = {k: None if v is None else v.detach() for k, v in R.items()}
    dO, dU = (d.double() * float(p) for d, p in zip((dout, du), parts))
    bound = ref.norm_bounds(dtype, *[D[k] for k in ("x", "h", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b")], kind, 1e-3, dO, dU)
    ref.within(out, OUT.detach(), bound["x_out"](OUT.detach()), "x_out")
    ref.within(u, UU.detach(), bound["u"](UU.detach()), "u")
    if not train:
        return
    names = [k for k, v in t.items() if v is not None]
    want = torch.autograd.grad([OUT, UU], [R[k] for k in names], [dO, dU])
    pick = [(o, d.cuda()) for o, d, p in zip((out, u), (dout, du), parts) if p]
    got = torch.autograd.grad([o for o, _ in pick], [dev[k] for k in names], [d for _, d in pick], allow_unused=True)
    for k, a, c in zip(names, got, want):
        if a is None:
            assert not c.any(), k
            continue
        ref.within(a, c, bound[k](c), k)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 8), (3, 7), (5, 64), (9, 512), (6, 513), (7, 1001), (5, 1024), (4, 2047), (3, 4096), (2, 8000), (3, 16384), (2, 10001), (2500, 64), (1100, 128), (300, 130), (70, 200), (2100, 16), (1030, 33), (600, 4104), (530, 8192), (300, 9000), (37, 1), (37, 3), (65, 5), (33, 63), (40, 129), (9, 4097), (600, 8191)])
def test_norm_sizes(ops, m, n, kind, dt):
    _check_norm(ops, m, n, 1, dt, kind, True, True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("m,n,groups", [(24, 96, 24), (24, 96, 8), (24, 96, 3), (24, 96, 1), (600, 40, 2), (1300, 24, 1300), (1030, 72, 10), (520, 600, 520)])
def test_norm_gates(ops, m, n, groups, kind, dt):
    _check_norm(ops, m, n, groups, dt, kind, True, True)


@pytest.mark.parametrize("gate,affine,parts", [(False, False, (True, True)), (False, True, (True, False)), (True, False, (False, True)), (True, True, (True, False))])
def test_norm_optional_arguments_and_gradients(ops, gate, affine, parts):
    _check_norm(ops, 20, 136, 4, "f32", "layer", gate, affine, parts=parts)


def test_norm_alone_forms_and_no_rows(ops):
    g = torch.Generator().manual_seed(8)
    x, w, b, du = _rand(g, 6, 4, 72, dtype=torch.float32), _rand(g, 72, dtype=torch.float32), _rand(g, 72, dtype=torch.float32), _rand(g, 6, 4, 72, dtype=torch.float32)
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    out, u = ops.residual_norm(xd, pre_weight=wd, pre_bias=bd)
    X, W, B = (t.double().requires_grad_() for t in (x, w, b))
    U_ = ref.norm(X.view(24, 72), W, B, "layer", 1e-3)
    bound = ref.norm_bounds(torch.float32, x.double().view(24, 72), None, None, None, None, None, w.double(), b.double(), "layer", 1e-3,
                            torch.zeros(24, 72).double(), du.double().view(24, 72))
    ref.within(u.view(24, 72), U_.detach(), bound["u"](U_.detach()))
    want = torch.autograd.grad(U_, (X, W, B), du.double().view(24, 72))
    got = torch.autograd.grad(u, (xd, wd, bd), du.cuda())
    for k, a, c in zip(("x", "pre_w", "pre_b"), got, want):
        ref.within(a.view(c.shape) if k == "x" else a, c if k != "x" else c, bound[k](c.view(24, 72) if k == "x" else c).view(c.shape), k)
    both, = torch.autograd.grad([*ops.residual_norm(xd)], xd, [du.cuda(), torch.zeros_like(u)])
    assert torch.equal(both.cpu(), du)                                       # the first output is x itself
    h = torch.randn(6, 4, 72, device="cuda")
    gate = torch.randn(6, 72, device="cuda")
    flat = ops.residual_norm(x.cuda().view(24, 72), h.view(24, 72), gate)
    for form in (gate, gate.view(6, 1, 72)):
        for a, c in zip(ops.residual_norm(x.cuda(), h, form), flat):
            assert torch.equal(a.view(24, 72), c)
    full = gate.view(6, 1, 72).expand(6, 4, 72)
    for a, c in zip(ops.residual_norm(x.cuda(), h, full), flat):
        assert torch.equal(a.view(24, 72), c)
    e = torch.zeros(0, 72, device="cuda", requires_grad=True)
    ww = torch.ones(72, device="cuda", requires_grad=True)
    o, u = ops.residual_norm(e, e, None, ww, pre_weight=ww)
    d, dw = torch.autograd.grad((o, u), (e, ww), (torch.zeros(0, 72, device="cuda"),) * 2)
    assert d.shape == (0, 72) and not dw.any()


def test_norm_constant_large_and_misaligned_rows(ops):
    """A constant row has no deviation (eps holds it); a large common offset does not cost the variance its digits; a row with NaN stays alone."""
    x = torch.full((3, 1000), 4096.0, device="cuda")
    _, u = ops.residual_norm(x)
    assert not u.any()
    g = torch.Generator().manual_seed(1)
    v = torch.randn(4, 1000, generator=g) + 1000.0
    _, u = ops.residual_norm(v.cuda())
    want = ref.norm(v.double(), None, None, "layer", 1e-3)
    assert float((u.cpu().double() - want).abs().max()) < 1000 * 64 * ref.U     # |v| / deviation times the count of roundings
    a, b = torch.randn(5, 1024, device="cuda"), torch.randn(5, 1024, device="cuda")
    base = ops.residual_norm(a, b)
    odd = torch.empty(5 * 1024 + 1, device="cuda")[1:].view(5, 1024).copy_(a)
    for p, q in zip(ops.residual_norm(odd, b), base):
        assert float((p - q).abs().max()) < 64 * ref.U * float(q.abs().max())
    b2 = b.clone()
    b2[2, 5] = float("nan")
    for p, q in zip(ops.residual_norm(a, b2), base):
        assert bool(torch.isnan(p[2]).all()) and torch.equal(p[[0, 1, 3, 4]], q[[0, 1, 3, 4]])


def test_norm_gradient_against_differences(ops):
    g = torch.Generator().manual_seed(6)
    m, n = 12, 100
    t = [_rand(g, m, n, dtype=torch.float32), _rand(g, m, n, dtype=torch.float32), _rand(g, 3, n, dtype=torch.float32)] + [_rand(g, n, dtype=torch.float32) for _ in range(5)]
    dev = [v.cuda().requires_grad_() for v in t]
    dO, dU = _rand(g, m, n, dtype=torch.float32), _rand(g, m, n, dtype=torch.float32)
    grads = torch.autograd.grad(ops.residual_norm(*dev, "layer", 1e-3), dev, (dO.cuda(), dU.cuda()))
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=g).double() * 1e-5

        def at(s):
            o, u = ref.residual_norm(*[v.double() + (s * d if q == i else 0) for q, v in enumerate(t)], "layer", 1e-3)
            return float((o * dO.double()).sum() + (u * dU.double()).sum())
        size = float((gr.double().cpu() * d).abs().sum())
        assert abs((at(1) - at(-1)) / 2 - float((gr.double().cpu() * d).sum())) < 1e-5 * size + 1e-8


# ------------------------------------------------------------------ together
def _block(ops, p, x, seed, counter=None):
    """A trunk of two residual blocks: norm, Dense + gelu, Dense + dropout, then the normalised step into the next block."""
    out, u = ops.residual_norm(x, pre_weight=p["n0w"], pre_bias=p["n0b"])
    for k in (1, 2):
        h = ops.dense(u, p[f"w{k}a"], p[f"b{k}a"], "gelu")
        h = ops.dense(h, p[f"w{k}b"], p[f"b{k}b"], None, None, 0.1, seed + k, 0, counter)
        out, u = ops.residual_norm(out, h, p["gate"], p[f"s{k}"], p[f"n{k}w"], p[f"n{k}b"], p["n0w"], p["n0b"])
    return ops.dropout(u, 0.2, seed, 0, out, counter)


def _params(g, d, f, groups, dtype):
    p = {"n0w": _rand(g, d, dtype=dtype, scale=0.1, shift=1.0), "n0b": _rand(g, d, dtype=dtype, scale=0.1), "gate": _rand(g, groups, d, dtype=dtype, scale=0.2, shift=1.0)}
    for k in (1, 2):
        p |= {f"w{k}a": _rand(g, d, f, dtype=dtype, scale=d ** -0.5), f"b{k}a": _rand(g, f, dtype=dtype, scale=0.1), f"w{k}b": _rand(g, f, d, dtype=dtype, scale=f ** -0.5),
              f"b{k}b": _rand(g, d, dtype=dtype, scale=0.1), f"s{k}": _rand(g, d, dtype=dtype, scale=0.1, shift=0.5),
              f"n{k}w": _rand(g, d, dtype=dtype, scale=0.1, shift=1.0), f"n{k}b": _rand(g, d, dtype=dtype, scale=0.1)}
    return p


def _block_ref(p, x, seed):
    kind, eps = "layer", 1e-3
    m, d = x.shape
    out, u = x, ref.norm(x, p["n0w"], p["n0b"], kind, eps)
    for k in (1, 2):
        h = ref.dense(u, p[f"w{k}a"], p[f"b{k}a"], "gelu")
        h = ref.dense(h, p[f"w{k}b"], p[f"b{k}b"], None, None, ref.keep_factor(m, d, 0.1, seed + k))
        out, u = ref.residual_norm(out, h, p["gate"], p[f"s{k}"], p[f"n{k}w"], p[f"n{k}b"], p["n0w"], p["n0b"], kind, eps)
    return u * ref.keep_factor(m, d, 0.2, seed) + out


@pytest.mark.parametrize("dt,tol", [("f32", 2e-5), ("bf16", 0.05)])
def test_a_trunk_of_all_three(ops, dt, tol):
    """Two blocks forward and backward: normwise, 30 roundings of a type deep with gains of order one (fp32 sums add a few 1e-7 each;
    in bf16 each of about ten layers adds 2^-8 or so of its own size, and so do their gradients on the way back)."""
    dtype = TYPES[dt]
    g = torch.Generator().manual_seed(12)
    m, d, f, groups = 96, 104, 264, 4
    p = _params(g, d, f, groups, dtype)
    x, dy = _rand(g, m, d, dtype=dtype), _rand(g, m, d, dtype=dtype)
    dev = {k: v.cuda().requires_grad_() for k, v in p.items()}
    xd = x.cuda().requires_grad_()
    y = _block(ops, dev, xd, 50)
    R = {k: v.double().requires_grad_() for k, v in p.items()}
    X = x.double().requires_grad_()
    Y = _block_ref(R, X, 50)
    got = torch.autograd.grad(y, [xd, *dev.values()], dy.cuda())
    want = torch.autograd.grad(Y, [X, *R.values()], dy.double())
    for name, a, c in zip(("y", "x", *p), (y.detach(), *got), (Y.detach(), *want)):
        err = float((a.double().cpu() - c).norm() / c.norm())
        assert err < tol, (name, err)


def test_same_bits_every_time_and_on_another_stream(ops):
    g = torch.Generator().manual_seed(13)
    p = {k: v.cuda().requires_grad_() for k, v in _params(g, 200, 520, 2, torch.bfloat16).items()}
    x, dy = torch.randn(640, 200, generator=g).bfloat16().cuda().requires_grad_(), torch.randn(640, 200, generator=g).bfloat16().cuda()
    runs = []
    side = torch.cuda.Stream()
    for k in range(4):
        with torch.cuda.stream(side if k & 1 else torch.cuda.current_stream()):
            torch.cuda.synchronize()
            y = _block(ops, p, x, 3)
            runs.append([y.detach(), *torch.autograd.grad(y, [x, *p.values()], dy)])
        torch.cuda.synchronize()
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_captured_training_pass_replays_with_fresh_numbers(ops):
    """Forward and backward captured once; each replay reads the advanced word and the new input; replays are interleaved with
    eager calls of the same operators and checked against them."""
    g = torch.Generator().manual_seed(14)
    p = {k: v.cuda() for k, v in _params(g, 96, 136, 3, torch.float32).items()}
    x, dy = torch.randn(48, 96, generator=g).cuda(), torch.randn(48, 96, generator=g).cuda()
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    names = list(p)

    def step(counter, x_in, params):
        leaves = [x_in.detach().requires_grad_(), *[params[k].detach().requires_grad_() for k in names]]
        y = _block(ops, dict(zip(names, leaves[1:])), leaves[0], 21, counter)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(count, x, p)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(count, x, p)
    seen = []
    for k in range(4):
        count.fill_(1000 * k)
        x.copy_(torch.randn(48, 96, generator=g))
        eager = [t.clone() for t in step(count, x, p)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), k
        again = step(count, x, p)
        assert all(torch.equal(a, b) for a, b in zip(again, eager)), k
        seen.append(outs[0].clone())
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.parametrize("dt,m,k,n", [("f32", 100, 640, 72), ("f32", 1, 6400, 100), ("f32", 1408, 1100, 1000), ("bf16", 300, 2048, 264), ("bf16", 301, 2047, 263)])
def test_two_captured_graphs_share_nothing(ops, dt, m, k, n):
    """The general product split, few rows, split fp32 terms, tiles with a split reduction, tiles of packed operands."""
    g = torch.Generator().manual_seed(15)
    x = torch.randn(m, k, generator=g).to(TYPES[dt]).cuda()
    w1, w2 = (torch.randn(k, n, generator=g).to(TYPES[dt]).cuda() for _ in range(2))
    want = ops.dense(x, w1, None, "gelu"), ops.dense(x, w2, None, "gelu")
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in (w1, w2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.dense(x, w, None, "gelu"))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_offsets_past_32_bits(ops, dt):
    """Tensors of more than 2^31 elements: their last rows come out as those of a call that holds only them.  The products pick single
    elements: exact, but for fp32 ones as three bf16 terms (2^-25 left out, and up to six roundings of 2^-24: 2^-21 covers them)."""
    t = ref.TYPES[dt]
    same = torch.equal if dt == "bf16" else lambda a, b: bool(((a - b).abs() <= b.abs() * 2.0 ** -21).all())  # noqa: E731
    rows, cols, last = (1 << 21) + 5, 1032, 7
    x = torch.empty(rows, cols, device="cuda", dtype=t).normal_()
    tail = x[-last:].clone()
    y = ops.dropout(x, 0.25, 3)
    assert torch.equal(y[-last:], ops.dropout(tail, 0.25, 3, rows - last))
    out, u = ops.residual_norm(x, y, kind="rms")
    alone = ops.residual_norm(tail, y[-last:].clone(), kind="rms")
    assert torch.equal(out[-last:], alone[0]) and torch.equal(u[-last:], alone[1])
    st = torch.ones(rows, 4, device="cuda")
    st[:, 0] = st[:, 2] = 0.0
    need = [True, True] + [False] * 6
    whole = ops.residual_norm_bwd(x, y, None, None, None, None, None, None, 1, 1, 1e-3, st, x, None, need)
    part = ops.residual_norm_bwd(tail, y[-last:].clone(), None, None, None, None, None, None, 1, 1, 1e-3, st[-last:].clone(), tail, None, need)
    assert torch.equal(whole[0][-last:], part[0]) and torch.equal(whole[1][-last:], part[1])
    del out, u, alone, whole, part, y, st
    # dx of a product whose dy is the large tensor, y of one whose y is, dw of one whose x is
    w = torch.zeros(8, cols, device="cuda", dtype=t)
    w[torch.arange(8), torch.arange(8) * 129] = 1.0
    small = torch.ones(rows, 8, device="cuda", dtype=t)
    dx = ops.dense_bwd(x, small, w, None, 0, 0.0, 0, 0, None, True, False, False)[0]
    assert same(dx[-last:], x[-last:, ::129][:, :8])
    y = ops.dense(dx, w)
    assert same(y[-last:, ::129][:, :8], dx[-last:]) and int((y[-last:] != 0).sum()) <= 8 * last
    del y, dx
    small.zero_()
    small[-1] = 1.0
    dw = ops.dense_bwd(small, x, torch.zeros(cols, 8, device="cuda", dtype=t), None, 0, 0.0, 0, 0, None, False, True, False)[1]
    assert torch.equal(dw, x[-1][:, None].expand(cols, 8))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("k,n", [(65544, 32776), (1024, 2100008), (65543, 32777)])
def test_weights_of_more_than_2_to_the_31_elements(ops, k, n, dt):
    """Rows of x with a single one pick rows of w, the last among them, on every path a forward call takes."""
    t = ref.TYPES[dt]
    w = torch.empty(k, n, device="cuda", dtype=t).normal_()
    for m in (1, 2, 5, 20):
        x = torch.zeros(m, k, device="cuda", dtype=t)
        at = k - 1 - torch.arange(m) * 3
        x[torch.arange(m), at] = 1.0
        assert torch.equal(ops.dense(x, w), w[at.cuda()])


def test_calls_from_several_threads_at_once(ops):
    """Each thread on a stream of its own: nothing is shared between calls, so each gets what it gets alone."""
    import threading

    def work(i):
        g = torch.Generator(device="cuda").manual_seed(i)
        m, k, n = [(1, 700, 264), (300, 264, 520), (129, 100, 77), (64, 1001, 333)][i % 4]
        t = [torch.float32, torch.bfloat16, torch.float16][i % 3]
        x, w, r = (torch.randn(*s, device="cuda", generator=g).to(t).requires_grad_() for s in ((m, k), (k, n), (m, n)))
        y = ops.dense(x, w, None, "gelu", r, 0.1, i)
        out, u = ops.residual_norm(r, y, kind="rms")
        return [y.detach(), u.detach()] + list(torch.autograd.grad((u * u).sum() + out.sum(), (x, w, r)))

    alone = [work(i) for i in range(8)]
    torch.cuda.synchronize()
    together = [None] * 8

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                together[i] = work(i)
        s.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, together):
        assert b is not None and all(torch.equal(p, q) for p, q in zip(a, b))
