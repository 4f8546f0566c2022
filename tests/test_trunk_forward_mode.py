"""Forward-mode derivatives of the dense-trunk operators: none are computed, so a dual tensor is refused, in the forward call and in
the backward pass, instead of counting as one without a tangent.  On the CPU with stand-ins for the kernels; on the GPU as it is."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(scope="module")
def ops():
    import vae_eeg_xai_amd.ops  # noqa: F401
    lib = torch.library.Library("veex", "IMPL")
    lib.impl("dense_fwd", lambda x, w, b, act, r, rate, seed, row, c, keep: (x @ w, x.new_empty(0)), "CPU")
    lib.impl("dense_bwd", lambda dy, x, w, pre, *a: (dy @ w.t(), x.t() @ dy, dy.sum(0)), "CPU")
    lib.impl("dropout_fwd", lambda x, rate, seed, row, r, c: 2 * x, "CPU")
    lib.impl("residual_norm_fwd", lambda x, h, *a: (x + h, x - h, x.new_zeros(x.shape[0], 4)), "CPU")
    lib.impl("residual_norm_bwd", lambda x, h, *a: [x.clone() if i < 2 else x.new_empty(0) for i in range(8)], "CPU")
    yield torch.ops.veex
    lib._destroy()


def _calls(ops, dev):
    """Each public op as a function of one of its tensors."""
    g = torch.Generator().manual_seed(1)
    x, w, b, r, row = (torch.randn(*s, generator=g).to(dev) for s in ((6, 8), (8, 4), (4,), (6, 4), (8,)))
    return {
        "dense x": (lambda t: ops.dense(t, w, b, "gelu"), x), "dense w": (lambda t: ops.dense(x, t), w),
        "dense bias": (lambda t: ops.dense(x, w, t), b), "dense residual": (lambda t: ops.dense(x, w, None, None, t), r),
        "dropout x": (lambda t: ops.dropout(t, 0.5, 1), x), "dropout residual": (lambda t: ops.dropout(x, 0.5, 1, 0, t), x),
        "norm x": (lambda t: ops.residual_norm(t, x)[1], x), "norm h": (lambda t: ops.residual_norm(x, t)[0], x),
        "norm gate": (lambda t: ops.residual_norm(x, x, t)[0], row), "norm scale": (lambda t: ops.residual_norm(x, x, None, t)[0], row),
        "norm pre_weight": (lambda t: ops.residual_norm(x, x, pre_weight=t)[1], row),
    }


NAMES = ["dense x", "dense w", "dense bias", "dense residual", "dropout x", "dropout residual", "norm x", "norm h", "norm gate", "norm scale", "norm pre_weight"]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_dual_inputs_are_refused(ops, name, dev):
    f, t = _calls(ops, dev)[name]
    for learns in (False, True):
        with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(fwad.make_dual(t.clone().requires_grad_(learns), torch.ones_like(t)))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jacfwd(f)(t)
    with fwad.dual_level():                       # without a tangent a call inside a dual level is an ordinary one
        assert f(t).numel() > 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", ["dense x", "dense w", "dropout x", "norm x", "norm h"])
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_dual_gradient_is_refused(ops, name, dev, create_graph):
    f, t = _calls(ops, dev)[name]
    t = t.clone().requires_grad_()
    y = f(t)
    with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(y, t, fwad.make_dual(torch.ones_like(y), torch.ones_like(y)), create_graph=create_graph)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_residual_passes_its_gradient_and_tangent_on(ops, dev):
    x, w = torch.ones(6, 8, device=dev), torch.ones(8, 4, device=dev)
    for f, shape in ((lambda t: ops.dense(x, w, None, None, t), (6, 4)), (lambda t: ops.dropout(x, 0.5, 1, 0, t), (6, 8))):
        r = torch.zeros(*shape, device=dev, requires_grad=True)
        y = f(r)
        dy, tangent = torch.randn_like(y), torch.randn_like(y)
        with fwad.dual_level():
            dr, = torch.autograd.grad(y, r, fwad.make_dual(dy, tangent))
            got = fwad.unpack_dual(dr)
            assert torch.equal(got.primal, dy) and torch.equal(got.tangent, tangent)
