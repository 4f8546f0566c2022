"""Operators of a dense trunk beside the convolution layers of ops.py: ``torch.ops.veex.dense``, ``dropout`` and
``residual_norm`` (include/veex.h: veex_dense_*, veex_dropout, veex_residual_norm_*).  Importing vae_eeg_xai_amd.ops registers them.

    dense(x, w, bias=None, activation=None, residual=None, rate=0.0, seed=0, first_row=0, counter=None) -> y
        y = residual + D(act(x w + bias));  x (..., K), w (K, N) as keras.layers.Dense keeps it (models.py:238-241,264),
        activation None | 'linear' | 'relu' | 'gelu' (erf) | 'silu' | 'sigmoid', D = dropout over y's rows and columns.
    dropout(x, rate, seed, first_row=0, residual=None, counter=None) -> y
        y = residual + keep x / (1 - rate), rate taken to the nearest 1/65536.
    residual_norm(x, h=None, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None,
                  kind='layer', eps=1e-3) -> (x_out, u)
        x_out = x + scale gate Norm(h; post), u = Norm(x_out; pre); without h: (x, Norm(x; pre)).  kind 'layer' or 'rms', up to
        16384 columns.  gate: one row of N for all of x ((N,)), one for each of x's leading indices ((B, N) or (B, 1, N) for
        x (B, T, N)), or x's shape; for a two-dimensional x also (G, N) with G dividing the rows, row r taking gate[r // (rows / G)].

float32, bfloat16 and float16, one type for all tensors of a call; sums and statistics are fp32 inside.  All are differentiable
once (dropout any number of times) in every tensor but ``counter``.

Dropout keeps no mask: the decision for an element is a function of (seed, first_row + counter + its row, its column), so forward
and backward draw the same one, and shards of a batch that pass their first global row draw what one process would.
``counter`` is an int64 word on the device that is read when the kernel runs: a captured step that advances it draws anew at
every replay.  The backward pass uses the word's value at the forward call.

Low level: a small Python entry picks the differentiable or the plain path and calls ``veex::dense_fwd`` etc., which are
registered for the ``cuda`` device type only, each with a fake implementation.  These are plain dispatcher registrations: a
training call of a small layer spends several times less on the host than through torch.library.custom_op.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "linear": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
_KINDS = {"layer": 0, "rms": 1}
_RELU = 1
MAX_COLS = 16384              # VEEX_NORM_MAX_COLS
_U64 = (1 << 64) - 1

_L = torch.library.Library("veex", "FRAGMENT")


def _p(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _on_device(fn):
    """Runs a launching function with its first tensor's device current (kernels go to the current device's stream)."""
    def call(x, *args):
        index = x.device.index
        if index == torch.cuda.current_device():
            return fn(x, *args)
        with torch.cuda.device(index):
            return fn(x, *args)
    return call


def _stream(x: Tensor):
    return torch._C._cuda_getCurrentRawStream(x.device.index)



def _contig(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _check_same(what: str, x: Tensor, **others: Optional[Tensor]) -> None:
    if x.dtype not in _TYPES:
        raise ValueError(f"{what}: float32, bfloat16 or float16 tensors, not {x.dtype}")
    for name, t in others.items():
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")


def _check_dropout(what: str, x: Tensor, rate: float, first_row: int, counter: Optional[Tensor]) -> None:
    if not 0.0 <= rate < 1.0 - 2.0 ** -17:
        raise ValueError(f"{what}: rate {rate} is outside [0, 1 - 2^-17)")
    if first_row < 0:
        raise ValueError(f"{what}: first_row is negative")
    if counter is not None and (counter.dtype != torch.int64 or counter.numel() != 1 or counter.device != x.device):
        raise ValueError(f"{what}: counter has to be one int64 word on x's device")


def _rows(x: Tensor) -> int:
    n = x.shape[-1]
    return x.numel() // n if n else 0


def _grads(*tensors: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------ dropout
_L.define("dropout_fwd(Tensor x, float rate, int seed, int first_row, Tensor? residual, Tensor? counter) -> Tensor")
_L.define("dropout(Tensor x, float rate, int seed, int first_row=0, Tensor? residual=None, Tensor? counter=None) -> Tensor")


@_on_device
def _dropout_cuda(x, rate, seed, first_row, residual, counter):
    x = _contig(x)
    residual = _contig(residual)
    y = torch.empty_like(x)
    if x.numel():
        check(lib.veex_dropout(_p(x), _p(residual), _p(y), _rows(x), x.shape[-1], _TYPES[x.dtype], rate, seed & _U64, first_row,
                               _p(counter), _stream(x)), "dropout")
    return y


_L.impl("dropout_fwd", _dropout_cuda, "CUDA")


@torch.library.register_fake("veex::dropout_fwd", lib=_L)
def _(x, rate, seed, first_row, residual, counter):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rate, seed, first_row, residual, counter):
        ctx.args = rate, seed, first_row
        # (the word as the forward call saw it: the caller may advance it before the backward pass)
        ctx.save_for_backward(counter + 0 if counter is not None and ctx.needs_input_grad[0] else None)
        return torch.ops.veex.dropout_fwd(x, rate, seed, first_row, residual, counter)

    @staticmethod
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            rate, seed, first_row = ctx.args
            dx = dropout(dy, rate, seed, first_row, None, ctx.saved_tensors[0])
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None, None


def dropout(x, rate, seed, first_row=0, residual=None, counter=None):
    _check_same("dropout", x, residual=residual)
    _check_dropout("dropout", x, rate, first_row, counter)
    if x.dim() < 1:
        raise ValueError("dropout: x has no columns")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"dropout: residual {tuple(residual.shape)} is not of x's shape {tuple(x.shape)}")
    if _grads(x, residual):
        return _Dropout.apply(x, rate, seed, first_row, residual, counter)
    return torch.ops.veex.dropout_fwd(x, rate, seed, first_row, residual, counter)


_L.impl("dropout", dropout, "CompositeImplicitAutograd")


# ------------------------------------------------------------------ dense
_L.define("dense_fwd(Tensor x, Tensor w, Tensor? bias, int activation, Tensor? residual, float rate, int seed, int first_row, "
          "Tensor? counter, bool keep) -> (Tensor, Tensor)")
_L.define("dense_bwd(Tensor dy, Tensor x, Tensor w, Tensor? pre, int activation, float rate, int seed, int first_row, "
          "Tensor? counter, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)")
_L.define("dense(Tensor x, Tensor w, Tensor? bias=None, str? activation=None, Tensor? residual=None, float rate=0.0, int seed=0, "
          "int first_row=0, Tensor? counter=None) -> Tensor")


def _as_rows(x: Tensor) -> Tensor:
    """x as (rows, K) with neighbouring columns next to each other: a view where its strides allow it."""
    k = x.shape[-1]
    x = x if x.dim() == 2 else x.reshape(-1, k)
    if x.shape[0] > 1 and (x.stride(1) != 1 and k > 1 or x.stride(0) < k) or x.shape[0] <= 1 and not x.is_contiguous():
        x = x.contiguous()
    return x


def _dense_desc(x2: Tensor, w: Tensor, activation, rate, seed, first_row, counter):
    d = _lib.DenseDesc()
    d.struct_size = C.sizeof(_lib.DenseDesc)
    d.x, d.w = x2.data_ptr(), w.data_ptr()
    d.rows, d.k, d.n = x2.shape[0], w.shape[0], w.shape[1]
    d.ldx = x2.stride(0) if d.rows > 1 else d.k
    d.dtype, d.activation = _TYPES[x2.dtype], activation
    d.rate, d.seed, d.first_row, d.counter = rate, seed & _U64, first_row, _p(counter)
    return d


def _workspace(nbytes: int, device, what: str) -> Optional[Tensor]:
    if nbytes < 0:
        check(-1, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


@_on_device
def _dense_cuda(x, w, bias, activation, residual, rate, seed, first_row, counter, keep):
    x2, w, bias, residual = _as_rows(x), _contig(w), _contig(bias), _contig(residual)
    y = torch.empty(*x.shape[:-1], w.shape[1], dtype=x.dtype, device=x.device)
    pre = torch.empty_like(y) if keep else torch.empty(0, dtype=x.dtype, device=x.device)
    d = _dense_desc(x2, w, activation, rate, seed, first_row, counter)
    d.bias, d.residual, d.y, d.pre = _p(bias), _p(residual), y.data_ptr(), pre.data_ptr() if keep else None
    if d.rows:
        ws = _workspace(lib.veex_dense_fwd_workspace_bytes(C.byref(d)), x.device, "dense")
        if ws is not None:
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.veex_dense_fwd(C.byref(d), _stream(x)), "dense")
    return y, pre


_L.impl("dense_fwd", _dense_cuda, "CUDA")


@torch.library.register_fake("veex::dense_fwd", lib=_L)
def _(x, w, bias, activation, residual, rate, seed, first_row, counter, keep):
    y = x.new_empty(*x.shape[:-1], w.shape[1])
    return y, torch.empty_like(y) if keep else x.new_empty(0)


@_on_device
def _dense_bwd_cuda(dy, x, w, pre, activation, rate, seed, first_row, counter, need_x, need_w, need_b):
    x2, wc, dy, pre = _as_rows(x), _contig(w), _contig(dy), _contig(pre)
    rows = x2.shape[0]
    make = torch.empty if rows else torch.zeros
    none = torch.empty(0, dtype=x.dtype, device=x.device)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else none
    dw = make(w.shape, dtype=x.dtype, device=x.device) if need_w else none
    db = make(w.shape[1], dtype=x.dtype, device=x.device) if need_b else none
    if rows and (need_x or need_w or need_b):
        d = _dense_desc(x2, wc, activation, rate, seed, first_row, counter)
        d.dy, d.pre = dy.data_ptr(), _p(pre)
        d.dx, d.dw, d.db = dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None, db.data_ptr() if need_b else None
        ws = _workspace(lib.veex_dense_bwd_workspace_bytes(C.byref(d)), x.device, "dense backward")
        if ws is not None:
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.veex_dense_bwd(C.byref(d), _stream(x)), "dense backward")
    return dx, dw, db


_L.impl("dense_bwd", _dense_bwd_cuda, "CUDA")


@torch.library.register_fake("veex::dense_bwd", lib=_L)
def _(dy, x, w, pre, activation, rate, seed, first_row, counter, need_x, need_w, need_b):
    none = x.new_empty(0)
    return (x.new_empty(x.shape) if need_x else none, x.new_empty(w.shape) if need_w else none,
            x.new_empty(w.shape[1]) if need_b else none)


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, activation, residual, rate, seed, first_row, counter):
        need = any(ctx.needs_input_grad[:3])
        # relu: y itself says where the gradient passes, unless a residual was added to it
        by_output = activation == _RELU and residual is None
        y, pre = torch.ops.veex.dense_fwd(x, w, bias, activation, residual, rate, seed, first_row, counter,
                                          need and activation != 0 and not by_output)
        ctx.args = activation, rate, seed, first_row
        if need:
            ctx.save_for_backward(x, w, None if activation == 0 else y if by_output else pre,
                                  counter + 0 if counter is not None and rate > 0.0 else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = dw = db = None
        if need_x or need_w or need_b:
            x, w, pre, counter = ctx.saved_tensors
            dx, dw, db = torch.ops.veex.dense_bwd(dy, x, w, pre, *ctx.args, counter, need_x, need_w, need_b)
        return (dx if need_x else None, dw if need_w else None, db if need_b else None, None,
                dy if ctx.needs_input_grad[4] else None, None, None, None, None)


def dense(x, w, bias=None, activation=None, residual=None, rate=0.0, seed=0, first_row=0, counter=None):
    _check_same("dense", x, w=w, bias=bias, residual=residual)
    _check_dropout("dense", x, rate, first_row, counter)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"dense: activation {activation!r} is none of {sorted(k for k in _ACTIVATIONS if k)}")
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[0] or 0 in w.shape:
        raise ValueError(f"dense: x {tuple(x.shape)} is not (..., K) for w {tuple(w.shape)} = (K, N) with K, N >= 1")
    n = w.shape[1]
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"dense: bias {tuple(bias.shape)} is not ({n},)")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"dense: residual {tuple(residual.shape)} is not of y's shape {(*x.shape[:-1], n)}")
    act = _ACTIVATIONS[activation]
    if _grads(x, w, bias, residual):
        return _Dense.apply(x, w, bias, act, residual, rate, seed, first_row, counter)
    return torch.ops.veex.dense_fwd(x, w, bias, act, residual, rate, seed, first_row, counter, False)[0]


_L.impl("dense", dense, "CompositeImplicitAutograd")


# ------------------------------------------------------------------ residual_norm
_NORM_ARGS = ("Tensor? h, Tensor? gate, Tensor? scale, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, "
              "Tensor? pre_bias, int groups, int kind, float eps")
_L.define(f"residual_norm_fwd(Tensor x, {_NORM_ARGS}, bool keep) -> (Tensor, Tensor, Tensor)")
_L.define(f"residual_norm_bwd(Tensor x, {_NORM_ARGS}, Tensor stats, Tensor? dx_out, Tensor? du, bool[] need) -> Tensor[]")
_L.define("residual_norm(Tensor x, Tensor? h=None, Tensor? gate=None, Tensor? scale=None, Tensor? post_weight=None, "
          "Tensor? post_bias=None, Tensor? pre_weight=None, Tensor? pre_bias=None, str kind='layer', float eps=0.001) -> (Tensor, Tensor)")


def _norm_desc(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps):
    d = _lib.ResidualNormDesc()
    d.struct_size = C.sizeof(_lib.ResidualNormDesc)
    d.x, d.h, d.gate, d.scale = x.data_ptr(), _p(h), _p(gate), _p(scale)
    d.post_w, d.post_b, d.pre_w, d.pre_b = _p(post_w), _p(post_b), _p(pre_w), _p(pre_b)
    d.rows, d.cols, d.groups = _rows(x), x.shape[-1], groups
    d.dtype, d.kind, d.eps = _TYPES[x.dtype], kind, eps
    return d


@_on_device
def _norm_cuda(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, keep):
    x, h, gate, scale, post_w, post_b, pre_w, pre_b = map(_contig, (x, h, gate, scale, post_w, post_b, pre_w, pre_b))
    none = torch.empty(0, dtype=x.dtype, device=x.device)
    out = torch.empty_like(x) if h is not None else none
    u = torch.empty_like(x)
    stats = torch.empty(_rows(x) if keep else 0, 4, dtype=torch.float32, device=x.device)
    if x.numel():
        d = _norm_desc(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps)
        d.x_out, d.u, d.stats = out.data_ptr() if h is not None else None, u.data_ptr(), stats.data_ptr() if keep else None
        check(lib.veex_residual_norm_fwd(C.byref(d), _stream(x)), "residual_norm")
    return out, u, stats


_L.impl("residual_norm_fwd", _norm_cuda, "CUDA")


@torch.library.register_fake("veex::residual_norm_fwd", lib=_L)
def _(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, keep):
    u = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = x.numel() // x.shape[-1]
    return (torch.empty_like(u) if h is not None else x.new_empty(0), u,
            x.new_empty(rows if keep else 0, 4, dtype=torch.float32))


@_on_device
def _norm_bwd_cuda(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, stats, dx_out, du, need):
    given = (x, h, gate, scale, post_w, post_b, pre_w, pre_b)
    x, h, gate, scale, post_w, post_b, pre_w, pre_b = map(_contig, given)
    dx_out, du = _contig(dx_out), _contig(du)
    rows = _rows(x)
    make = torch.empty if rows else torch.zeros
    none = torch.empty(0, dtype=x.dtype, device=x.device)
    grads = [make(t.shape, dtype=x.dtype, device=x.device) if n else none for t, n in zip(given, need)]
    if rows:
        d = _norm_desc(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps)
        d.stats, d.dx_out, d.du = stats.data_ptr(), _p(dx_out), _p(du)
        for field, g, n in zip(("dx", "dh", "dgate", "dscale", "dpost_w", "dpost_b", "dpre_w", "dpre_b"), grads, need):
            setattr(d, field, g.data_ptr() if n else None)
        floats = lib.veex_residual_norm_bwd_workspace_floats(rows, x.shape[-1], groups)
        ws = torch.empty(floats, dtype=torch.float32, device=x.device)
        d.workspace, d.workspace_floats = ws.data_ptr(), floats
        check(lib.veex_residual_norm_bwd(C.byref(d), _stream(x)), "residual_norm backward")
    return grads


_L.impl("residual_norm_bwd", _norm_bwd_cuda, "CUDA")


@torch.library.register_fake("veex::residual_norm_bwd", lib=_L)
def _(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, stats, dx_out, du, need):
    return [x.new_empty(t.shape) if n else x.new_empty(0) for t, n in zip((x, h, gate, scale, post_w, post_b, pre_w, pre_b), need)]


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps):
        ctx.set_materialize_grads(False)
        out, u, stats = torch.ops.veex.residual_norm_fwd(x, h, gate, scale, post_w, post_b, pre_w, pre_b, groups, kind, eps, True)
        ctx.save_for_backward(x, h, gate, scale, post_w, post_b, pre_w, pre_b, stats)
        ctx.args = groups, kind, eps
        return (out, u) if h is not None else u

    @staticmethod
    @once_differentiable
    def backward(ctx, *douts):
        dx_out, du = douts if len(douts) == 2 else (None, douts[0])
        need = list(ctx.needs_input_grad[:8])
        if dx_out is None and du is None:
            return (None,) * 11
        *given, stats = ctx.saved_tensors
        grads = torch.ops.veex.residual_norm_bwd(*given, *ctx.args, stats, dx_out, du, need)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def _gate_groups(gate: Tensor, x: Tensor) -> int:
    """Rows of the gate: its leading indices are the first ones of x's, those left out (or 1) share a gate."""
    lead, rows = list(gate.shape[:-1]), _rows(x)
    groups = _rows(gate)
    while lead and lead[-1] == 1:
        lead.pop()
    fits = len(lead) < x.dim() and lead == list(x.shape[:len(lead)])
    if not fits and x.dim() == 2 and len(lead) == 1:
        fits = lead[0] > 0 and rows % lead[0] == 0
    if gate.dim() < 1 or gate.shape[-1] != x.shape[-1] or not fits:
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} does not go with x {tuple(x.shape)}")
    return max(groups, 1)


def residual_norm(x, h=None, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None,
                  kind="layer", eps=1e-3) -> Tuple[Tensor, Tensor]:
    _check_same("residual_norm", x, h=h, gate=gate, scale=scale, post_weight=post_weight, post_bias=post_bias,
                pre_weight=pre_weight, pre_bias=pre_bias)
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: kind {kind!r} is neither 'layer' nor 'rms'")
    if not eps >= 0.0:
        raise ValueError("residual_norm: eps has to be >= 0")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"residual_norm: rows of 1 to {MAX_COLS} columns, not x {tuple(x.shape)}")
    if h is None and any(t is not None for t in (gate, scale, post_weight, post_bias)):
        raise ValueError("residual_norm: gate, scale and the post norm's parameters go with h")
    if h is not None and h.shape != x.shape:
        raise ValueError(f"residual_norm: h {tuple(h.shape)} is not of x's shape {tuple(x.shape)}")
    for name, t in (("scale", scale), ("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight),
                    ("pre_bias", pre_bias)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"residual_norm: {name} {tuple(t.shape)} is not ({x.shape[-1]},)")
    groups = 1 if gate is None else _gate_groups(gate, x)
    args = (x, h, gate, scale, post_weight, post_bias, pre_weight, pre_bias, groups, _KINDS[kind], eps)
    if _grads(*args[:8]):
        res = _ResidualNorm.apply(*args)
        return res if h is not None else (x, res)
    out, u, _ = torch.ops.veex.residual_norm_fwd(*args, False)
    return (out, u) if h is not None else (x, u)


_L.impl("residual_norm", residual_norm, "CompositeImplicitAutograd")
