"""CPU: what the dense-trunk operators refuse, their fake implementations, their C-ABI's host side, and the 64-bit
restatement the GPU tests compare with (known answers of the generator; gradients against differences).  No kernel is launched."""
import ctypes as C

import pytest
import torch

import trunk_ref as ref


@pytest.fixture(scope="module", autouse=True)
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    return torch.ops.veex


def test_generator_known_answers():
    """The published vectors of philox4x32-10: all-zero, all-one, and the digits of pi."""
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = ref.philox([[c] for c in ctr], key)
        assert tuple(int(g[0]) for g in got) == want


def test_dropout_numbers_are_fair_and_follow_rows():
    f = ref.keep_factor(400, 500, 0.3, 99)
    assert abs(float((f == 0).double().mean()) - 0.3) < 5 * (0.3 * 0.7 / 200000) ** 0.5
    assert torch.equal(ref.keep_factor(10, 500, 0.3, 99, first_row=390), f[390:])
    assert torch.equal(ref.keep_factor(400, 77, 0.3, 99), f[:, :77])


@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu", "sigmoid"])
def test_reference_dense_gradients_against_differences(act):
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (7, 6), (6,), (5, 6), (5, 6)))
    f = ref.keep_factor(5, 6, 0.25, 3)
    for k, v in enumerate((x, w, b, r)):
        v.requires_grad_()
        y = ref.dense(x, w, b, act, r, f)
        gr = torch.autograd.grad((y * dy).sum(), v)[0]
        v = v.detach()
        d = torch.randn(v.shape, generator=g, dtype=torch.float64) * 1e-5
        at = lambda s: float((ref.dense(*[(u.detach() + s * d if i == k else u.detach()) for i, u in enumerate((x, w, b))], act,  # noqa: E731
                                        r.detach() + (s * d if k == 3 else 0.0), f) * dy).sum())
        assert abs((at(1) - at(-1)) / 2 - float((gr * d).sum())) < 1e-9


@pytest.mark.parametrize("bad,message", [
    (lambda o, t: o.dense(t(2, 3), t(4, 5)), "K, N"),
    (lambda o, t: o.dense(t(2, 3), t(3, 0)), "K, N"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), t(5)), "bias"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), t(1, 4)), "bias"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, "tanh"), "activation"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, t(1, 4)), "residual"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4).bfloat16()), "w is"),
    (lambda o, t: o.dense(t(2, 3).double(), t(3, 4).double()), "float32, bfloat16 or float16"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, None, 1.0), "rate"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, None, -0.1), "rate"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, None, float("nan")), "rate"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, None, 0.5, 1, -1), "first_row"),
    (lambda o, t: o.dense(t(2, 3), t(3, 4), None, None, None, 0.5, 1, 0, t(1)), "counter"),
    (lambda o, t: o.dropout(t(2, 3), 0.999999, 1), "rate"),
    (lambda o, t: o.dropout(t(2, 3), 0.5, 1, 0, t(2, 4)), "residual"),
    (lambda o, t: o.dropout(t(2, 3), 0.5, 1, 0, None, torch.zeros(2, dtype=torch.int64)), "counter"),
    (lambda o, t: o.dropout(t(2, 3).long(), 0.5, 1), "float32, bfloat16 or float16"),
    (lambda o, t: o.residual_norm(t(2, 3), kind="batch"), "kind"),
    (lambda o, t: o.residual_norm(t(2, 3), eps=-1.0), "eps"),
    (lambda o, t: o.residual_norm(t(2, 16385)), "columns"),
    (lambda o, t: o.residual_norm(t(2, 3), t(2, 4)), "h ("),
    (lambda o, t: o.residual_norm(t(2, 3), None, t(3)), "go with h"),
    (lambda o, t: o.residual_norm(t(6, 3), t(6, 3), t(4, 3)), "gate"),
    (lambda o, t: o.residual_norm(t(6, 3), t(6, 3), t(6, 1)), "gate"),
    (lambda o, t: o.residual_norm(t(2, 4, 3), t(2, 4, 3), t(1, 4, 3)), "gate"),
    (lambda o, t: o.residual_norm(t(2, 4, 3), t(2, 4, 3), t(4, 3)), "gate"),
    (lambda o, t: o.residual_norm(t(6, 3), t(6, 3), None, t(1, 3)), "scale"),
    (lambda o, t: o.residual_norm(t(6, 3), pre_weight=t(4)), "pre_weight"),
])
def test_refusals(ops, bad, message):
    with pytest.raises(ValueError) as e:
        bad(ops, lambda *s: torch.zeros(*s))
    assert message in str(e.value)


def test_cpu_tensors_have_no_kernel(ops):
    x = torch.zeros(2, 8)
    for call in (lambda: ops.dense(x, torch.zeros(8, 4)), lambda: ops.dropout(x, 0.5, 1), lambda: ops.residual_norm(x, x)):
        with pytest.raises(NotImplementedError):
            call()


def test_fake_tensors(ops):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 5, 6, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(6, 8, device="cuda", dtype=torch.bfloat16)
        y = ops.dense(x, w, None, "gelu", None, 0.1, 7)
        assert y.shape == (2, 5, 8) and y.dtype == torch.bfloat16
        dx, dw, db = ops.dense_bwd(y, x, w, y, 2, 0.1, 7, 0, None, True, True, False)
        assert dx.shape == x.shape and dw.shape == w.shape and db.numel() == 0
        assert ops.dropout(x, 0.5, 1, 0, x).shape == x.shape
        out, u = ops.residual_norm(x, x, torch.empty(2, 1, 6, device="cuda", dtype=torch.bfloat16))
        assert out.shape == x.shape and u.shape == x.shape
        out, u = ops.residual_norm(x, kind="rms")
        assert out is x and u.shape == x.shape
        assert ops.residual_norm_fwd(x, x, None, None, None, None, None, None, 1, 0, 1e-3, True)[2].shape == (10, 4)


def test_descriptors_match_the_header():
    from vae_eeg_xai_amd._lib import DenseDesc, ResidualNormDesc
    assert C.sizeof(DenseDesc) == 11 * 8 + 3 * 8 + 4 * 4 + 8 + 2 * 8 + 8 + 2 * 4
    assert C.sizeof(ResidualNormDesc) == 22 * 8 + 8 + 2 * 8 + 4 * 4 + 2 * 4


def test_host_side_refuses_before_any_launch():
    from vae_eeg_xai_amd import _lib
    lib = _lib.lib
    err = lambda: lib.veex_last_error().decode()  # noqa: E731
    some = 1 << 20                       # never dereferenced: every call below is refused on the host
    assert lib.veex_dropout(None, None, some, 4, 8, 0, 0.5, 1, 0, None, None) == -1 and "x and y" in err()
    assert lib.veex_dropout(some, None, some, -1, 8, 0, 0.5, 1, 0, None, None) == -1
    assert lib.veex_dropout(some, None, some, 4, 0, 0, 0.5, 1, 0, None, None) == -1
    assert lib.veex_dropout(some, None, some, 4, 8, 3, 0.5, 1, 0, None, None) == -1
    assert lib.veex_dropout(some, None, some, 4, 8, 0, 1.0, 1, 0, None, None) == -1 and "rate" in err()
    assert lib.veex_dropout(some, None, some, 4, 8, 0, float("nan"), 1, 0, None, None) == -1
    assert lib.veex_dropout(some, None, some, 0, 8, 0, 0.5, 1, 0, None, None) == 0          # nothing to do
    d = _lib.DenseDesc()
    d.struct_size = C.sizeof(d)
    d.rows, d.k, d.n, d.ldx = 512, 6400, 100, 6400
    need = lib.veex_dense_fwd_workspace_bytes(C.byref(d))
    assert need > 0 and lib.veex_dense_bwd_workspace_bytes(C.byref(d)) > 0
    d.x = d.w = d.y = some
    assert lib.veex_dense_fwd(C.byref(d), None) == -2 and str(need) in err()
    d.workspace, d.workspace_bytes = some, need - 1
    assert lib.veex_dense_fwd(C.byref(d), None) == -2
    assert lib.veex_dense_bwd(C.byref(d), None) == -1 and "dy" in err()
    for field, value in (("rows", -1), ("k", 0), ("n", 0), ("ldx", 6399), ("dtype", 5), ("activation", 9), ("rate", 1.0), ("struct_size", 8)):
        e = _lib.DenseDesc.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.veex_dense_fwd_workspace_bytes(C.byref(e)) == -1, field
        assert lib.veex_dense_fwd(C.byref(e), None) == -1, field
    q = _lib.ResidualNormDesc()
    q.struct_size = C.sizeof(q)
    q.rows, q.cols, q.groups, q.eps = 12, 64, 1, 1e-3
    assert lib.veex_residual_norm_fwd(C.byref(q), None) == -1 and "x and u" in err()
    q.x = q.u = some
    q.h = some
    assert lib.veex_residual_norm_fwd(C.byref(q), None) == -1                                # h without x_out
    q.x_out = q.gate = some
    for field, value in (("groups", 5), ("groups", 0), ("cols", 0), ("cols", 16385), ("kind", 2), ("dtype", -1), ("eps", -1.0), ("struct_size", 4)):
        e = _lib.ResidualNormDesc.from_buffer_copy(q)
        setattr(e, field, value)
        assert lib.veex_residual_norm_fwd(C.byref(e), None) == -1, field
    assert lib.veex_residual_norm_bwd(C.byref(q), None) == -1                                # no stats, no workspace
    floats = lib.veex_residual_norm_bwd_workspace_floats(12, 64, 1)
    assert floats >= 5 * 64 and lib.veex_residual_norm_bwd_workspace_floats(12, 64, 5) == -1
    q.stats = q.workspace = some
    q.workspace_floats = floats - 1
    assert lib.veex_residual_norm_bwd(C.byref(q), None) == -2 and "workspace" in err()


def test_more_blocks_than_a_launch_takes_are_refused():
    from vae_eeg_xai_amd import _lib
    lib = _lib.lib
    some = 1 << 20                       # never dereferenced
    for dtype, rows, k, n in ((0, 1 << 31, 1, 64), (0, 1, 1, 1 << 30), (1, 1 << 31, 512, 256)):
        d = _lib.DenseDesc()
        d.struct_size = C.sizeof(d)
        d.rows, d.k, d.n, d.ldx, d.dtype = rows, k, n, k, dtype
        d.x = d.w = d.y = d.workspace = some
        d.workspace_bytes = 1 << 62
        assert lib.veex_dense_fwd(C.byref(d), None) == -1 and "tiles" in lib.veex_last_error().decode()
    q = _lib.ResidualNormDesc()
    q.struct_size = C.sizeof(q)
    q.rows, q.cols, q.groups, q.eps = 1 << 24, 8, 1 << 23, 1e-3
    q.x = q.h = q.gate = q.dgate = q.du = q.dx = q.workspace = some
    q.stats = some + 4
    q.workspace_floats = 1 << 60
    assert lib.veex_residual_norm_bwd(C.byref(q), None) == -1 and "aligned" in lib.veex_last_error().decode()
    q.stats = some
    assert lib.veex_residual_norm_bwd(C.byref(q), None) == -1 and "groups" in lib.veex_last_error().decode()
    q.u = q.x_out = some
    q.stats = some + 8
    assert lib.veex_residual_norm_fwd(C.byref(q), None) == -1 and "aligned" in lib.veex_last_error().decode()
