"""How the row operators are called, without a GPU: what of it does not depend on a kernel's result."""
import pytest
import torch

from artifact_amd import rof_module
from artifact_amd._lib import RofError
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
