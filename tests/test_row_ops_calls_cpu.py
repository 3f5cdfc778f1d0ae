"""How the row operators are called, without a GPU: what of it does not depend on a kernel's result."""
import pytest
import torch

from artifact_amd import _lib, rof_module
from artifact_amd._lib import RofError
from artifact_amd.ROF_models import ROF_GCN, ROF_GIN
from artifact_amd.row_ops import ROF_DropoutState


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm_backward", "dropout", "dropout_state_next"])
def test_the_operators_are_the_dispatchers(name):
    """What records a program from the calls it sees (torch.jit.trace, make_fx) sees nothing else of a compiled function than
    what it asks PyTorch for: the allocation of its result."""
    rof_module.row_operators()
    assert torch._C._dispatch_has_kernel_for_dispatch_key(f"rof::{name}", "CUDA")
    schema = getattr(torch.ops.rof, name).default._schema
    assert schema.is_mutable == (name == "dropout_state_next")


def test_the_state_does_not_move_on_during_a_backward_pass():
    class AsACheckpoint(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, grad):
            ROF_DropoutState(3).next(2)
            return grad

    x = torch.ones(3, requires_grad=True)
    with pytest.raises(RofError, match="backward pass"):
        AsACheckpoint.apply(x).sum().backward()


class Times(torch.nn.Module):
    """A convolution's place in a model, without a graph or a GPU."""

    def __init__(self, factor):
        super().__init__()
        self.factor = factor

    def forward(self, x, info):
        return x * self.factor


def model_without_graph(cls=ROF_GCN, layers=2, rate=0.4, **kw):
    kw = {"activation": torch.tanh} | kw
    model = cls(6, 6, 6, layers if cls is ROF_GCN else layers + 1, dropout=rate, **kw)
    model.layers = torch.nn.ModuleList(Times(2.0) for _ in range(layers + 1))
    return model


@pytest.mark.parametrize("cls", [ROF_GCN, ROF_GIN])
def test_a_model_pickled_before_norms_and_states_still_runs(cls):
    model = model_without_graph(cls).eval()
    x = torch.linspace(-1, 1, 12).reshape(2, 6)
    want = model(x, None)
    for name in ("norms", "dropout_state"):      # what such an object does not have
        del model.__dict__[name]
    assert torch.equal(model(x, None), want) and torch.equal(want, torch.tanh(torch.tanh(x * 2) * 2) * 2)


def test_a_replaced_norm_or_dropout_is_called_by_itself():
    x = torch.linspace(-1, 1, 12).reshape(2, 6) ** 3
    model = model_without_graph(activation=torch.relu, norm="layer", rate=0.0)
    model.norms = torch.nn.ModuleList(torch.nn.LayerNorm(6) for _ in range(2))
    want = torch.nn.functional.layer_norm
    assert torch.equal(model(x, None), torch.relu(want(torch.relu(want(x * 2, (6,))) * 2, (6,))) * 2)
    seen = []

    class Mine(torch.nn.Module):
        def forward(self, h):
            seen.append(h)
            return h + 1

    for norm in (None, "layer"):
        model = model_without_graph(norm=norm, dropout_seed=3)       # a state on the CPU: nothing may ask it for values
        if norm:
            model.norms = torch.nn.ModuleList(torch.nn.Identity() for _ in range(2))
        model.dropout = Mine()
        assert torch.equal(model(x, None), (torch.tanh((torch.tanh(x * 2) + 1) * 2) + 1) * 2)
        assert len(seen) == 2 and torch.equal(seen[0], torch.tanh(x * 2))
        seen.clear()


@pytest.mark.parametrize("f,n", [(512, 399997), (300, 1599985), (256, 399997), (47, 1599985), (5, 12799873), (1, 25599745)])
def test_the_workspace_grows_where_the_launch_becomes_tiles(f, n):
    """From 100000 rounds of rows on, which are 4 to 256 rows by width and type: n is the first such number of rows in the type
    with fewer rows a round.  Before that a row per workgroup that can stay, 1280."""
    size = _lib.lib().rof_layer_norm_backward_workspace_bytes
    assert size(100000, f) == size(n - 1, f) == 1280 * 2 * f * 4
    assert size(n, f) == (16384 + 128) * 2 * f * 4
