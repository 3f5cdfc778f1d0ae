"""Norm and counter-based dropout inside the models (ROF_GCN, ROF_GIN, the training command): a training step against a
dense float64 reference with the same masks, the passes against the operators they are made of, and the default models
unchanged."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import torch.nn.functional as F                                         # noqa: E402

from artifact_amd.graphgen import features, make_workload               # noqa: E402
from artifact_amd.reuse_conv import build_input_info                    # noqa: E402
from artifact_amd.ROF_models import ROF_GCN, ROF_GIN                    # noqa: E402
from artifact_amd.row_ops import dropout, layer_norm                    # noqa: E402
from row_oracle import kept, scale                                      # noqa: E402

DEV = "cuda"


@pytest.fixture(scope="module")
def graph():
    ip, ix = make_workload("c1", 5)                                      # 512 nodes, self loops: every degree >= 1
    n = len(ip) - 1
    a = torch.zeros((n, n), dtype=torch.float64)
    a[torch.from_numpy(np.repeat(np.arange(n), np.diff(ip))), torch.from_numpy(ix.astype(np.int64))] = 1.0
    r = torch.from_numpy(1.0 / np.sqrt(np.diff(ip).astype(np.float64)))
    return ip, ix, a, r[:, None] * a * r[None, :], build_input_info(ip, ix, 3, device=DEV, min_consumers=2)


def _gcn(info, kernel_type="ROF_v2", layers=2, activation=F.relu, rate=0.4, **kw):
    torch.manual_seed(5)
    model = ROF_GCN(24, 20, 5, layers, activation, rate, add_self_loops=False, reuse_size=info.reuse_size,
                    kernel_type=kernel_type, **kw).to(DEV)
    with torch.no_grad():
        for layer in model.layers:
            layer.bias.uniform_(-0.3, 0.3)
        for norm in model.norms or []:
            norm.weight.uniform_(0.5, 1.5)
            norm.bias.uniform_(-0.3, 0.3)
    return model


def _norm64(h, weight, bias, eps=1e-5):
    c = h - h.mean(1, keepdim=True)
    return c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * weight + bias


def _compare(model, loss, ref_loss, ref):
    """Gradients within 2e-4 in the 2-norm: every operator of a step is held to 1e-5 by its own tests, a hidden layer is
    five of them forward and backward, and the norm magnifies what comes in by 1 / (the rows' spread), up to 4 here."""
    assert abs(loss.item() - ref_loss.item()) <= 2e-4 * abs(ref_loss.item())
    loss.backward()
    ref_loss.backward()
    got = {k: p.grad for k, p in model.named_parameters() if p.grad is not None}
    assert set(got) == set(ref)
    for k, p in ref.items():
        diff = (got[k].cpu().double() - p.grad).norm().item()
        assert diff <= 2e-4 * p.grad.norm().item(), f"{k}: {diff / p.grad.norm().item():.2e}"


@pytest.mark.parametrize("kernel_type", ["GNNA", "ROF_v1", "ROF_v2"])
@pytest.mark.parametrize("norm,seed", [("layer", 77), ("layer", None), (None, 77)])
def test_a_gcn_training_step_matches_dense_float64(graph, kernel_type, norm, seed):
    ip, ix, _, a_hat, info = graph
    n, rate = len(ip) - 1, 0.4 if seed is not None else 0.0              # torch's own masks have no reference
    model = _gcn(info, kernel_type, rate=rate, norm=norm, dropout_seed=seed)
    x, y = torch.from_numpy(features(n, 24, seed=41)), torch.arange(n) % 5
    loss = F.cross_entropy(model(x.to(DEV), info), y.to(DEV))
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.named_parameters()
         if "part_result_cache" not in k}
    h = x.double()
    for i in range(3):
        h = a_hat @ (h @ p[f"layers.{i}.weight"]) + p[f"layers.{i}.bias"]
        if i < 2:
            if norm:
                h = _norm64(h, p[f"norms.{i}.weight"], p[f"norms.{i}.bias"])
            h = torch.relu(h)
            if rate:
                h = h * torch.from_numpy(kept(np.arange(n), 20, rate, seed, i)) * scale(rate)
    _compare(model, loss, F.cross_entropy(h, y), p)


@pytest.mark.parametrize("norm", ["layer", None])
def test_a_gin_training_step_matches_dense_float64(graph, norm):
    ip, ix, a, _, info = graph
    n, seed, rate = len(ip) - 1, 5, 0.3
    torch.manual_seed(6)
    model = ROF_GIN(24, 20, 5, 3, dropout=rate, eps=0.1, norm=norm, dropout_seed=seed).to(DEV)
    x, y = torch.from_numpy(features(n, 24, seed=43)) * 0.05, torch.arange(n) % 5
    loss = F.cross_entropy(model(x.to(DEV), info), y.to(DEV))
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.named_parameters()}
    h = x.double()
    for i in range(3):
        h = (1.1 * h + a @ h) @ p[f"layers.{i}.mlp.weight"].t() + p[f"layers.{i}.mlp.bias"]
        if i < 2:
            if norm:
                h = _norm64(h, p[f"norms.{i}.weight"], p[f"norms.{i}.bias"])
            h = torch.relu(h) * torch.from_numpy(kept(np.arange(n), 20, rate, seed, i)) * scale(rate)
    _compare(model, loss, F.cross_entropy(h, y), p)


@pytest.mark.parametrize("compute_dtype", [None, "bf16"])
@pytest.mark.parametrize("activation", [F.relu, torch.tanh, None])
@pytest.mark.parametrize("norm,seed", [("layer", 3), ("layer", None), (None, 3)])
def test_the_models_passes_are_the_operators(graph, activation, norm, seed, compute_dtype):
    """Layer by layer through the operators' functions: the same bits, whichever of them the model runs in one pass."""
    ip, ix, _, _, info = graph
    model = _gcn(info, activation=activation, norm=norm, dropout_seed=seed, compute_dtype=compute_dtype)
    x = torch.from_numpy(features(len(ip) - 1, 24, seed=44)).to(DEV)
    torch.manual_seed(9)
    got = model(x, info)
    torch.manual_seed(9)
    h, rng = x, None if seed is None else torch.tensor([seed, 0], device=DEV)
    for i, layer in enumerate(model.layers):
        h = layer(h, info)
        if i == 2:
            break
        if norm:
            m = model.norms[i]
            if activation is not torch.tanh:
                h = layer_norm(h, m.weight, m.bias, relu=activation is not None, dropout=0.4 if seed is not None else 0.0,
                               rng=rng, call=i)
            else:
                h = torch.tanh(layer_norm(h, m.weight, m.bias))
        elif activation is not None and not model._fused_act:
            h = activation(h)
        if seed is None:
            h = F.dropout(h, 0.4)
        elif not norm or activation is torch.tanh:
            h = dropout(h, 0.4, rng, call=i)
    assert torch.equal(got, h) and got.dtype == torch.float32
    if seed is not None:
        assert model.dropout_state.state.tolist() == [3, 2]
        model.eval()
        model(x, info)
        assert model.dropout_state.state.tolist() == [3, 2]


def test_a_resumed_model_draws_the_masks_of_the_uninterrupted_one(graph):
    ip, ix, _, _, info = graph
    x = torch.from_numpy(features(len(ip) - 1, 24, seed=44)).to(DEV)
    model = _gcn(info, norm="layer", dropout_seed=8)
    first = model(x, info)
    saved = {k: v.clone() for k, v in model.state_dict().items()}
    second, third = model(x, info), model(x, info)
    assert not torch.equal(first, second)
    other = _gcn(info, norm="layer", dropout_seed=99)
    other.load_state_dict(saved)
    assert torch.equal(other(x, info), second) and torch.equal(other(x, info), third)


@pytest.mark.parametrize("activation", [F.relu, torch.tanh])
def test_the_models_without_the_new_arguments_are_what_they_were(graph, activation):
    ip, ix, _, _, info = graph
    x = torch.from_numpy(features(len(ip) - 1, 24, seed=44)).to(DEV)
    for model in (_gcn(info, activation=activation), ROF_GIN(24, 20, 5, 3, activation=activation, dropout=0.4).to(DEV)):
        assert not any(k.startswith(("norms", "dropout")) for k in model.state_dict())
        assert isinstance(model.dropout, torch.nn.Dropout) and model.dropout.p == 0.4
        torch.manual_seed(3)
        got = model(x, info)
        torch.manual_seed(3)
        h = x
        for i, layer in enumerate(model.layers):
            if i != 0:
                h = F.dropout(h, 0.4)
            h = layer(h, info)
            if i != 2 and not getattr(model, "_fused_act", False):
                h = activation(h)
        assert torch.equal(got, h)


def test_the_training_command_runs_with_them(monkeypatch, capsys):
    from artifact_amd import train as command

    monkeypatch.setattr(sys, "argv", ["train", "--workload", "c1", "--scale-down", "3", "--epochs", "4", "--norm", "layer",
                                      "--dropout_seed", "7"])
    command.main()
    assert "mean epoch" in capsys.readouterr().out
