"""Operators on the feature rows between two graph convolutions, through librof.so (include/rof.h): layer norm with the
ReLU and the dropout of a hidden layer in the same pass, and dropout whose mask is computed and never stored.

Not upstream: its models put torch's dropout on the input of every layer but the first (ROF_evaluation/ROF_main.py:192-200)
and do not normalise.  `layer_norm` and `dropout` are differentiable functions of 2-D tensors with one row per node,
`ROF_LayerNorm`, `ROF_Dropout` and `ROF_DropoutState` the modules that `ROF_GCN` and `ROF_GIN` are built from.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import DropoutOpts, RofError, check
from .layout import ROF_BF16, ROF_F32

__all__ = ["layer_norm", "dropout", "ROF_LayerNorm", "ROF_Dropout", "ROF_DropoutState"]

LAYER_NORM_MAX_COLUMNS = 16384   # ROF_LAYER_NORM_MAX_COLUMNS of include/rof.h
_TYPES = {torch.float32: ROF_F32, torch.bfloat16: ROF_BF16}


def _rows(name, t):
    """A matrix the kernels take: 2-D, float32 or bfloat16, on a GPU, unit column stride, rows that do not overlap."""
    if not t.is_cuda or t.dim() != 2 or t.dtype not in _TYPES:
        raise RofError(f"{name} must be a 2-D float32 or bfloat16 CUDA tensor")
    if t.shape[1] == 0:
        raise RofError(f"{name} must have at least one column")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise RofError(f"{name} must have unit column stride and rows that do not overlap")


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _gradient(grad, like):
    """An incoming gradient as rows the kernels take (autograd hands over broadcast and transposed ones as well)."""
    if grad.dtype != like:
        grad = grad.to(like)
    ok = (grad.shape[1] == 1 or grad.stride(1) == 1) and (grad.shape[0] <= 1 or grad.stride(0) >= grad.shape[1])
    return grad if ok else grad.contiguous()


def _rate(p):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RofError("a dropout rate must lie between 0 and 1")
    return p


def _check_rng(rng, device):
    if rng is None:
        raise RofError("dropout needs rng: an int64 tensor {seed, offset} on the device of x (see ROF_DropoutState)")
    if rng.dtype != torch.int64 or rng.device != device or rng.numel() != 2 or not rng.is_contiguous():
        raise RofError("rng must be a contiguous int64 tensor of two elements {seed, offset} on the device of x")


def _check_param(name, t, x):
    if t is not None and (t.dtype != torch.float32 or t.device != x.device or t.dim() != 1 or t.numel() != x.shape[1]
                          or not t.is_contiguous()):
        raise RofError(f"{name} must be a contiguous float32 vector with one element per column on the device of x")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _drop_opts(p, rng, call):
    return C.byref(DropoutOpts(p, rng.data_ptr(), call)) if p else None


def _run_dropout(x, p, rng, call):
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        check(_lib.lib().rof_dropout(x.data_ptr(), _TYPES[x.dtype], _ld(x), x.shape[0], x.shape[1], out.data_ptr(), x.shape[1],
                                     C.byref(DropoutOpts(p, _ptr(rng), call)), _stream()))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, call):
        ctx.save_for_backward(rng)
        ctx.p, ctx.call, ctx.dtype = p, call, x.dtype
        return _run_dropout(x, p, rng, call)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _run_dropout(_gradient(grad, ctx.dtype), ctx.p, ctx.saved_tensors[0], ctx.call), None, None, None


def dropout(x, p, rng, call=0):
    """x with every element dropped with probability p (to the nearest multiple of 2^-16) and the others scaled by
    1 / (1 - p).  rng: int64 tensor {seed, offset} on the device; the mask is a function of it, of `call`, and of the
    element's row, column and number of columns, and is computed again for the gradient.  Modifying rng in place between
    the forward and the backward pass is an error: take the values of a step from ROF_DropoutState.next()."""
    _rows("x", x)
    p = _rate(p)
    _check_rng(rng, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, p, rng, int(call))
    return _run_dropout(x, p, rng, int(call))


def _run_norm(x, weight, bias, eps, relu, p, rng, call, out_dtype):
    n, f = x.shape
    out = torch.empty((n, f), dtype=out_dtype, device=x.device)
    with torch.cuda.device(x.device):
        check(_lib.lib().rof_layer_norm(x.data_ptr(), _TYPES[x.dtype], _ld(x), n, f, _ptr(weight), _ptr(bias), eps, relu,
                                        _drop_opts(p, rng, call), out.data_ptr(), _TYPES[out_dtype], f, _stream()))
    return out


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, relu, p, rng, call, out_dtype):
        ctx.save_for_backward(x, weight, bias, rng)
        ctx.args = (eps, relu, p, call, out_dtype)
        return _run_norm(x, weight, bias, eps, relu, p, rng, call, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, bias, rng = ctx.saved_tensors
        eps, relu, p, call, out_dtype = ctx.args
        n, f = x.shape
        grad = _gradient(grad, out_dtype)
        dx = torch.empty((n, f), dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(f, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[1] else None
        db = torch.empty(f, dtype=torch.float32, device=x.device) if ctx.needs_input_grad[2] else None
        L = _lib.lib()
        ws, nbytes = None, 0
        if dw is not None or db is not None:
            nbytes = L.rof_layer_norm_backward_workspace_bytes(n, f)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        with torch.cuda.device(x.device):
            check(L.rof_layer_norm_backward(grad.data_ptr(), _TYPES[out_dtype], _ld(grad), x.data_ptr(), _TYPES[x.dtype],
                                            _ld(x), n, f, _ptr(weight), _ptr(bias), eps, relu, _drop_opts(p, rng, call),
                                            _ptr(dx), f, _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream()))
        return dx, dw, db, None, None, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False, dropout=0.0, rng=None, call=0, out_dtype=None):
    """dropout(relu(layer norm of every row of x)) in one pass each way.

    x: [n, f] float32 or bfloat16, f <= 16384; weight, bias: float32 [f] or None (1 and 0); `relu` and `dropout` (a rate;
    rng and call as in `dropout`) are left out by default; out_dtype: float32 or bfloat16, by default x's.  Sums are taken
    in float32 and the result is rounded once.  The backward pass keeps x only and computes statistics, gate and mask from
    it again; its sums over rows have a fixed order, so the gradients are bitwise repeatable."""
    _rows("x", x)
    if x.shape[1] > LAYER_NORM_MAX_COLUMNS:
        raise RofError(f"layer_norm takes at most {LAYER_NORM_MAX_COLUMNS} columns")
    _check_param("weight", weight, x)
    _check_param("bias", bias, x)
    eps = float(eps)
    if not 0.0 <= eps <= 1e30:
        raise RofError("eps must not be negative")
    p = _rate(dropout)
    if p:
        _check_rng(rng, x.device)
    else:
        rng = None
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _TYPES:
        raise RofError("out_dtype must be float32 or bfloat16")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, bool(relu), p, rng, int(call), out_dtype)
    return _run_norm(x, weight, bias, eps, bool(relu), p, rng, int(call), out_dtype)


class ROF_DropoutState(torch.nn.Module):
    """The generator of a model's dropout layers: seed and offset on the device, as a buffer (saved and restored with the
    model, so that a resumed run draws the masks that the interrupted one would have).  `next(calls)` returns the values of
    one step and moves the offset on by `calls`; both happen on the device, so a captured step draws new masks whenever it
    is replayed.  Ranks that train together need seeds of their own."""

    def __init__(self, seed):
        super().__init__()
        self.register_buffer("state", torch.tensor([int(seed), 0], dtype=torch.int64))

    def next(self, calls=1):
        state = self.state
        if not state.is_cuda:
            raise RofError("the dropout state must be on the GPU (move the module there)")
        used = torch.empty_like(state)
        with torch.cuda.device(state.device):
            check(_lib.lib().rof_dropout_state_next(state.data_ptr(), int(calls), used.data_ptr(), _stream()))
        torch.autograd.graph.increment_version(state)
        return used


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

    def forward(self, x, rng=None, call=0, out_dtype=None):
        return layer_norm(x, self.weight, self.bias, eps=self.eps, relu=self.relu, dropout=self.p if self.training else 0.0,
                          rng=rng, call=call, out_dtype=out_dtype)

    def extra_repr(self):
        return f"{self.num_features}, eps={self.eps}, relu={self.relu}, dropout={self.p}"
