"""Models on top of the reuse-aware layers: counterpart of the upstream `ROF_models` module, which its
drivers import (`from ROF_models import ROF_GCN, ROF_inputInfo`, ROF_evaluation/ROF_main.py:31) but which is
not part of the upstream tree.  The constructor and call conventions are the ones the call sites fix:

    ROF_GCN(in_feats, n_hidden, n_classes, n_layers, activation, dropout, add_self_loops, reuse_size, kernel_type)
        (ROF_main.py:192-200, cuda/middle-rof.py:474-482)
    model(features, inputInfo)                (ROF_main.py:230)
    model(features, edge_index, inputInfo)    (cuda/middle-rof.py:496; edge_index is unused by the layers)

`n_layers` hidden convolutions plus the output convolution, i.e. n_layers + 1 layers (ROF_main.py:256 reports
"layers": n_layers + 1), activation between them, dropout on the input of every layer but the first.

Both models take two keyword arguments that upstream does not have:
    norm="layer"        layer norm of every hidden layer's output, before its activation
    dropout_seed=int    dropout from a counter-based generator whose mask is never stored (row_ops.dropout) in place of
                        torch.nn.Dropout; the generator's state is a buffer of the model
With both and a ReLU (or no activation), norm, activation and dropout of a hidden layer are one pass over its rows each way.
It is the norm that is called for it, so its hooks and wrappers take part, and its output is that of the whole pass.  A norm
that was replaced by another module, or given a ReLU or a dropout of its own, and a dropout that was replaced or has hooks,
run by themselves.
A forward pass with dropout_seed moves the model's state on, so it cannot be run again for its own backward pass
(activation checkpointing of the whole model): that raises RofError.
"""
from __future__ import annotations

import torch

from .reuse_conv import ROF_GCNConv, ROF_GINConv, ROF_inputInfo  # noqa: F401  (re-exported like upstream)
from .row_ops import ROF_Dropout, ROF_DropoutState, ROF_LayerNorm

__all__ = ["ROF_GCN", "ROF_GIN", "ROF_inputInfo"]

_RELUS = (torch.relu, torch.nn.functional.relu)


def _add_tails(model, widths, activation, rate, norm, dropout_seed):
    """What follows the hidden layers of these widths: the model's norms, activation, dropout and dropout state."""
    if norm not in (None, "layer"):
        raise ValueError("norm must be None or 'layer'")
    model.activation = activation
    model.norms = None if norm is None else torch.nn.ModuleList(ROF_LayerNorm(w) for w in widths)
    model.dropout = torch.nn.Dropout(p=rate) if dropout_seed is None else ROF_Dropout(rate)
    model.dropout_state = None if dropout_seed is None else ROF_DropoutState(dropout_seed)


def _takes_more(norm):
    """Whether the pass of this norm may hold the model's activation and dropout as well."""
    return type(norm).forward is ROF_LayerNorm.forward and not norm.relu and not norm.p


def _can_be_part(dropout):
    """Whether this dropout may run inside the pass of a norm: not one with hooks or a wrapper, which would not be called there."""
    return type(dropout).forward is ROF_Dropout.forward and not (
        "forward" in vars(dropout) or dropout._forward_hooks or dropout._forward_pre_hooks or dropout._backward_hooks or dropout._backward_pre_hooks)


def _run_layers(model, h, inputInfo, activated):
    """The layers and what is between them.  `activated`: the hidden layers apply the activation themselves."""
    last = len(model.layers) - 1
    # a model that was pickled whole before it could have them has neither
    norms, state = getattr(model, "norms", None), getattr(model, "dropout_state", None)
    counted = state is not None and isinstance(model.dropout, ROF_Dropout)
    rate = model.dropout.p if counted and model.dropout.training else 0.0
    # the values of this forward pass; norms that drop by themselves use the calls behind the model's own
    own = norms is not None and any(isinstance(norm, ROF_LayerNorm) and norm.p and norm.training for norm in norms)
    rng = state.next(2 * last if own else last) if state is not None and (rate or own) and last else None
    dropped = True                                                      # what the next layer reads is ready for it
    for i, layer in enumerate(model.layers):
        if not dropped:
            h = model.dropout(h, rng, call=i - 1) if counted else model.dropout(h)
        h = layer(h, inputInfo)
        if i == last:
            break
        dropped = False
        activation = None if activated else model.activation
        if norms is not None:
            norm, whole = norms[i], activation is None or activation in _RELUS
            if _takes_more(norm):
                dropped = whole and counted and _can_be_part(model.dropout)
                h = norm(h, rng, call=i, relu=whole and activation is not None, dropout=rate if dropped else 0.0)
                activation = None if whole else activation
            elif isinstance(norm, ROF_LayerNorm):
                h = norm(h, rng, call=last + i)
            else:
                h = norm(h)
        if activation is not None:
            h = activation(h)
    return h


class ROF_GCN(torch.nn.Module):
    def __init__(self, in_feats, n_hidden, n_classes, n_layers, activation, dropout, add_self_loops=False,
                 reuse_size=0, kernel_type="ROF_v1", bias=True, order="update_first", fuse_epilogue=True,
                 compute_dtype=None, norm=None, dropout_seed=None):
        """`order`, `fuse_epilogue` and `compute_dtype` are passed to every ROF_GCNConv (not upstream).  A ReLU
        activation is then applied by the aggregation kernel of each hidden layer rather than as a pass of its
        own.  compute_dtype="bf16": bfloat16 rows and GEMM operands, fp32 sums and parameters; hidden layers hand
        bfloat16 to each other, the last layer returns float32.  `norm`, `dropout_seed`: see the module."""
        super().__init__()
        dims = [in_feats] + [n_hidden] * n_layers + [n_classes]
        last = len(dims) - 2
        bf16 = compute_dtype in ("bf16", torch.bfloat16)
        self._fused_act = norm is None and bool(fuse_epilogue) and (kernel_type != "ROF_v1" or bf16) and activation in _RELUS
        self.layers = torch.nn.ModuleList(
            ROF_GCNConv(dims[i], dims[i + 1], bias=bias, add_self_loops=add_self_loops, reuse_size=reuse_size,
                        kernel_type=kernel_type, order=order, fuse_epilogue=fuse_epilogue,
                        activation="relu" if self._fused_act and i != last else None, compute_dtype=compute_dtype,
                        out_dtype="bf16" if bf16 and i != last else None)
            for i in range(len(dims) - 1))
        _add_tails(self, dims[1:-1], activation, dropout, norm, dropout_seed)

    def forward(self, features, *args):
        return _run_layers(self, features, args[-1], self._fused_act)


class ROF_GIN(torch.nn.Module):
    """GIN with sum aggregation (eps fixed) and one linear map per layer, e.g. 3 x (64 -> 64).  `norm`, `dropout_seed`:
    see the module."""

    def __init__(self, in_feats, n_hidden, n_classes, n_layers, activation=torch.relu, dropout=0.0, eps=0.0,
                 kernel_type="ROF_v2", norm=None, dropout_seed=None):
        super().__init__()
        dims = [in_feats] + [n_hidden] * (n_layers - 1) + [n_classes]
        self.layers = torch.nn.ModuleList(ROF_GINConv(dims[i], dims[i + 1], eps=eps, kernel_type=kernel_type)
                                          for i in range(len(dims) - 1))
        _add_tails(self, dims[1:-1], activation, dropout, norm, dropout_seed)

    def forward(self, features, *args):
        return _run_layers(self, features, args[-1], False)
