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

float32, bfloat16 and float16, one type for all tensors of a call; sums and statistics are fp32 inside.  In 16-bit types dense
rounds two more things than its results: z = x w + bias is kept for the backward pass in the type, as separate layers would keep
it, and dz = D'(dy) act'(z) goes into the products dx = dz w^T and dw = x^T dz in it (their error is that of two roundings, 1.4 times
that of one; db sums the unrounded dz).  Large float32 products are made of bf16 terms, to float32's rounding; operands below about
1e-33 keep fewer bits there.  A gate that learns has fewer than 2^22 rows, or one for each row of x.

All are differentiable
once (dropout any number of times) in every tensor but ``counter``, in reverse mode: a tensor with a forward-mode tangent
(torch.func.jvp, forward_ad.make_dual) is refused with NotImplementedError.

Dropout keeps no mask: the decision for an element is a function of (seed, first_row + counter + its row, its column), so forward
and backward draw the same one, and shards of a batch that pass their first global row draw what one process would.
``counter`` is an int64 word on the device that is read when the kernel runs: a captured step that advances it draws anew at
every replay.  The backward pass uses the word's value at the forward call.

dense takes an x whose rows lie any distance apart as it is; other tensors that are not contiguous, a transposed w among them, are
copied first, on every call.  All ops can be captured into graphs, training steps too.  As with every torch op, no eager
graph of the same leaves may be alive while a backward pass is captured: torch keeps a leaf's gradient node on the stream where
it was made, and the capture fails there.

The ops, their checks and their autograd are C++ (csrc/torch_ops.cpp, libveex_torch.so); this module loads them and adds the fake
implementations of the low-level ops ``veex::dense_fwd`` etc., whose kernels are registered for the ``cuda`` device type only.
"""
from __future__ import annotations

import os

import torch

from . import _lib

LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libveex_torch.so")
if not os.path.exists(LIB_PATH):
    raise _lib.VeexError(f"{LIB_PATH} not found: the torch extension is not built (run __graft_entry__.build()). There is no CPU fallback.")
torch.ops.load_library(LIB_PATH)


@torch.library.register_fake("veex::dropout_fwd")
def _(x, rate, seed, first_row, residual, counter):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.register_fake("veex::dense_fwd")
def _(x, w, bias, activation, residual, rate, seed, first_row, counter, keep):
    y = x.new_empty(*x.shape[:-1], w.shape[1])
    return y, torch.empty_like(y) if keep else x.new_empty(0)


@torch.library.register_fake("veex::dense_bwd")
def _(dy, x, w, pre, activation, rate, seed, first_row, counter, need_x, need_w, need_b):
    none = x.new_empty(0)
    return (x.new_empty(x.shape) if need_x else none, w.new_empty(w.shape) if need_w else none.clone(),
            x.new_empty(w.shape[1]) if need_b else none.clone())


@torch.library.register_fake("veex::residual_norm_fwd")
def _(x, h, gate, scale, post_weight, post_bias, pre_weight, pre_bias, groups, kind, eps, keep):
    u = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = x.numel() // x.shape[-1]
    return (torch.empty_like(u) if h is not None else x.new_empty(0), u,
            x.new_empty(rows if keep else 0, 4, dtype=torch.float32))


@torch.library.register_fake("veex::residual_norm_bwd")
def _(x, h, gate, scale, post_weight, post_bias, pre_weight, pre_bias, groups, kind, eps, stats, dx_out, du, need):
    given = (x, h, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    return [x.new_empty(t.shape) if n and t is not None else x.new_empty(0) for t, n in zip(given, need)]
