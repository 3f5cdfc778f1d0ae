"""Operators on the feature rows between two graph convolutions, through librof.so (include/rof.h): layer norm with the
ReLU and the dropout of a hidden layer in the same pass, and dropout whose mask is computed and never stored.

Not upstream: its models put torch's dropout on the input of every layer but the first (ROF_evaluation/ROF_main.py:192-200)
and do not normalise.  `layer_norm` and `dropout` are differentiable functions of 2-D tensors with one row per node,
`ROF_LayerNorm`, `ROF_Dropout` and `ROF_DropoutState` the modules that `ROF_GCN` and `ROF_GIN` are built from.  They are
operators of PyTorch's dispatcher (rof::layer_norm, rof::layer_norm_backward, rof::dropout, rof::dropout_state_next), so
torch.jit.trace and make_fx record them as calls; a traced program that is loaded in another process needs
`rof_module.row_operators()` called there first.  torch.func's transforms are refused.
"""
from __future__ import annotations

import torch

from . import rof_module
from ._lib import RofError

__all__ = ["layer_norm", "dropout", "ROF_LayerNorm", "ROF_Dropout", "ROF_DropoutState"]

_ops = None


def _compiled():
    global _ops
    if _ops is None:
        _ops = rof_module.row_operators()
    return _ops


def dropout(x, p, rng, call=0):
    """x with every element dropped with probability p (to the nearest multiple of 2^-16) and the others scaled by
    1 / (1 - p).

    x: 2-D float32 or bfloat16 CUDA tensor with unit column stride (rows may be apart).  rng: int64 tensor {seed, offset}
    on its device; the mask is a function of it, of `call`, and of the element's row, column and number of columns, and is
    computed again for the gradient.  Modifying rng in place between the forward and the backward pass is an error: take
    the values of a step from ROF_DropoutState.next().  Raises RofError for what it does not take."""
    return _compiled().dropout(x, p, rng, call)


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False, dropout=0.0, rng=None, call=0, out_dtype=None):
    """dropout(relu(layer norm of every row of x)) in one pass each way.

    x: [n, f] float32 or bfloat16 with unit column stride (rows may be apart), f <= 8192 or 16384; weight, bias: float32 [f]
    or None (1 and 0); `relu` and `dropout` (a rate; rng and call as in `dropout`) are left out by default; out_dtype: float32
    or bfloat16, by default x's.  Sums are taken in float32 and the result is rounded once.  The backward pass keeps x only
    and computes statistics, gate and mask from it again; its sums over rows have a fixed order, so the gradients are
    bitwise repeatable.  There is no second derivative.  Raises RofError for what it does not take."""
    return _compiled().layer_norm(x, weight, bias, eps, relu, dropout, rng, call, out_dtype)


def _rate(p):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RofError("a dropout rate must lie between 0 and 1")
    return p


class ROF_DropoutState(torch.nn.Module):
    """The generator of a model's dropout layers: seed and offset on the device, as a buffer (saved and restored with the
    model, so that a resumed run draws the masks that the interrupted one would have).  `next(calls)` returns the values of
    one step and moves the offset on by `calls`; both happen on the device, so a captured step draws new masks whenever it
    is replayed.  Ranks that train together need seeds of their own (and no broadcast of buffers).  A checkpointed function
    must be given the values, not call `next` itself: its second pass would draw other masks, so `next` raises RofError
    during a backward pass."""

    def __init__(self, seed):
        super().__init__()
        self.register_buffer("state", torch.tensor([int(seed), 0], dtype=torch.int64))

    def next(self, calls=1):
        return _compiled().dropout_state_next(self.state, calls)


class ROF_Dropout(torch.nn.Module):
    """torch.nn.Dropout's counterpart: `dropout` while training, the identity in evaluation and at rate 0."""

    def __init__(self, p=0.5):
        super().__init__()
        self.p = _rate(p)

    def forward(self, x, rng, call=0):
        return dropout(x, self.p, rng, call) if self.training and self.p else x

    def extra_repr(self):
        return f"p={self.p}"


class ROF_LayerNorm(torch.nn.Module):
    """Layer norm over the features of a node, with the ReLU and the dropout that may follow it in the same pass.
    Parameters are float32 whatever the type of the rows, as in the convolutions."""

    def __init__(self, num_features, eps=1e-5, elementwise_affine=True, bias=True, relu=False, dropout=0.0):
        super().__init__()
        self.num_features = int(num_features)
        self.eps = float(eps)
        self.relu = bool(relu)
        self.p = _rate(dropout)
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.empty(self.num_features))
        else:
            self.register_parameter("weight", None)
        if elementwise_affine and bias:
            self.bias = torch.nn.Parameter(torch.empty(self.num_features))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.weight is not None:
            torch.nn.init.ones_(self.weight)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, x, rng=None, call=0, out_dtype=None, relu=None, dropout=None):
        """`relu` and `dropout` (a rate, whatever the mode), where given, stand for the module's own."""
        if dropout is None:
            dropout = self.p if self.training else 0.0
        return layer_norm(x, self.weight, self.bias, eps=self.eps, relu=self.relu if relu is None else relu, dropout=dropout,
                          rng=rng, call=call, out_dtype=out_dtype)

    def extra_repr(self):
        return f"{self.num_features}, eps={self.eps}, relu={self.relu}, dropout={self.p}"
