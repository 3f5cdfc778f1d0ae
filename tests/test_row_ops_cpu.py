"""Row operators without a GPU: the oracle they are tested against, the checks of the C ABI (which answer before anything is
launched), and the refusals of the Python layer."""
import ctypes as C

import numpy as np
import pytest
import torch

from artifact_amd import _lib, row_ops
from artifact_amd._lib import DropoutOpts, RofError
from row_oracle import Norm, kept, philox, scale, threshold

ARG, UNSUPPORTED, WORKSPACE = -1, -6, -7
F32, BF16 = 0, 1
PTR = 1 << 20          # never dereferenced: every call below is refused on the host


@pytest.mark.parametrize("counter,key,rounds,words", [
    (0, 0, 10, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    (0xFFFFFFFF, 0xFFFFFFFF, 10, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    (0, 0, 7, (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
])
def test_the_oracles_generator_gives_the_published_vectors(counter, key, rounds, words):
    got = philox(np.full((1, 4), counter, dtype=np.uint64), (key, key), rounds)[0]
    assert tuple(int(v) for v in got) == words


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -17, 0.1, 0.5, 0.9, 1.0])
def test_the_oracles_mask_drops_at_the_rate(p):
    n, f = 500, 40
    mask = kept(np.arange(n), f, p, seed=7, offset=3)
    rate, t = 1.0 - mask.mean(), threshold(p) / 65536
    assert abs(rate - t) <= 6 * np.sqrt(max(t * (1 - t), 1e-12) / (n * f))     # six standard deviations
    assert abs(t - p) <= 2.0 ** -17
    assert t in (0.0, 1.0) or scale(p) * (1 - t) == pytest.approx(1.0)


def test_masks_of_other_seeds_offsets_and_rows_are_others():
    a = kept(np.arange(64), 64, 0.5, 1, 0)
    for b in (kept(np.arange(64), 64, 0.5, 2, 0), kept(np.arange(64), 64, 0.5, 1, 1), kept(np.arange(64, 128), 64, 0.5, 1, 0),
              kept(np.arange(64), 64, 0.5, 1 << 40, 0), kept(np.arange(64), 64, 0.5, 1, 1 << 40)):
        assert 0.4 < (a == b).mean() < 0.6       # 4096 fair coins: 0.5 within 0.1 (12 standard deviations)
    assert np.array_equal(a, kept(np.arange(64), 64, 0.5, 1, 2 ** 64))


@pytest.mark.parametrize("relu,p", [(False, 0.0), (True, 0.25)])
def test_the_oracles_gradient_is_the_difference_quotient(relu, p):
    rng = np.random.default_rng(3)
    n, f, step = 5, 11, 1e-6
    x, dy = rng.standard_normal((n, f)), rng.standard_normal((n, f))
    w, b = 1 + 0.3 * rng.standard_normal(f), 0.3 * rng.standard_normal(f)
    keep = kept(np.arange(n), f, p, 5, 1) if p else None

    def loss(x, w, b):
        return (Norm(x, w, b, relu=relu, keep=keep, p=p).y * dy).sum()

    (dx, dw, db), _ = Norm(x, w, b, relu=relu, keep=keep, p=p).backward(dy)
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        args = [x, w, b]
        for i in np.ndindex(grad.shape):
            e = np.zeros_like(args[at])
            e[i] = step
            up, down = list(args), list(args)
            up[at], down[at] = args[at] + e, args[at] - e
            # central difference: step^2 of curvature, 1e-16 / step of rounding
            assert (loss(*up) - loss(*down)) / (2 * step) == pytest.approx(grad[i], abs=1e-7)


def _norm(x=PTR, xt=F32, ldx=8, n=3, f=8, w=PTR, b=PTR, eps=1e-5, drop=None, out=PTR, ot=F32, ldo=8):
    return _lib.lib().rof_layer_norm(x, xt, ldx, n, f, w, b, eps, 0, drop, out, ot, ldo, None)


@pytest.mark.parametrize("args,code", [
    (dict(n=-1), ARG), (dict(f=0, ldx=0), ARG), (dict(ldx=7), ARG), (dict(ldo=7), ARG), (dict(x=None), ARG),
    (dict(out=None), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(eps=float("inf")), ARG),
    (dict(xt=2), UNSUPPORTED), (dict(ot=-1), UNSUPPORTED), (dict(f=8193, ldx=8193, ldo=8193), UNSUPPORTED),
    (dict(xt=BF16, f=16385, ldx=16385, ldo=16385), UNSUPPORTED),
    (dict(x=PTR + 2), ARG), (dict(xt=BF16, x=PTR + 1), ARG), (dict(w=PTR + 2), ARG), (dict(b=PTR + 1), ARG),
    (dict(out=PTR + 2), ARG), (dict(ot=BF16, out=PTR + 1), ARG),
    (dict(drop=DropoutOpts(-0.1, PTR, 0)), ARG), (dict(drop=DropoutOpts(1.5, PTR, 0)), ARG),
    (dict(drop=DropoutOpts(float("nan"), PTR, 0)), ARG), (dict(drop=DropoutOpts(0.5, None, 0)), ARG),
    (dict(drop=DropoutOpts(0.5, PTR + 4, 0)), ARG), (dict(n=0, x=None, out=None), 0),
])
def test_layer_norm_refuses_what_it_cannot_run(args, code):
    if isinstance(args.get("drop"), DropoutOpts):
        args = args | {"drop": C.byref(args["drop"])}
    assert _norm(**args) == code


@pytest.mark.parametrize("args,code", [
    (dict(dout=None), ARG), (dict(ldd=7), ARG), (dict(dout=PTR + 2), ARG), (dict(lddx=7), ARG), (dict(dx=PTR + 1), ARG),
    (dict(dw=PTR + 2), ARG), (dict(db=PTR + 2), ARG), (dict(ws=None), WORKSPACE), (dict(size=3 * 2 * 8 * 4 - 1), WORKSPACE),
    (dict(ws=PTR + 8), WORKSPACE), (dict(f=8193, ldx=8193), UNSUPPORTED), (dict(dt=7), UNSUPPORTED), (dict(n=-1), ARG),
    (dict(dx=None, dw=None, db=None, ws=None, size=0), 0),      # nothing wanted: nothing launched
])
def test_layer_norm_backward_refuses_what_it_cannot_run(args, code):
    a = dict(dout=PTR, dt=F32, ldd=8, x=PTR, xt=F32, ldx=8, n=3, f=8, dx=PTR, lddx=8, dw=PTR, db=PTR, ws=PTR, size=1 << 20) | args
    assert _lib.lib().rof_layer_norm_backward(a["dout"], a["dt"], a["ldd"], a["x"], a["xt"], a["ldx"], a["n"], a["f"], PTR, PTR,
                                              1e-5, 0, None, a["dx"], a["lddx"], a["dw"], a["db"], a["ws"], a["size"],
                                              None) == code


def test_backward_workspace_holds_a_row_per_workgroup():
    size = _lib.lib().rof_layer_norm_backward_workspace_bytes
    assert size(0, 8) == 0 and size(5, 0) == 0
    assert size(3, 8) == 3 * 2 * 8 * 4
    assert size(1280, 47) == size(99999, 47) == 1280 * 2 * 47 * 4
    assert size(10 ** 7, 47) == (16384 + 128) * 2 * 47 * 4 and size(10 ** 7, 512) == (16384 + 128) * 2 * 512 * 4
    assert size(10 ** 7, 513) == 1280 * 2 * 513 * 4


@pytest.mark.parametrize("args,code", [
    (dict(x=None), ARG), (dict(out=None), ARG), (dict(ldx=7), ARG), (dict(ldo=7), ARG), (dict(n=-1), ARG), (dict(f=0), ARG),
    (dict(t=3), UNSUPPORTED), (dict(x=PTR + 2), ARG), (dict(out=PTR + 1), ARG), (dict(drop=DropoutOpts(2.0, PTR, 0)), ARG),
    (dict(drop=DropoutOpts(0.5, None, 0)), ARG), (dict(n=0), 0), (dict(no=True), ARG),
])
def test_dropout_refuses_what_it_cannot_run(args, code):
    a = dict(x=PTR, t=F32, ldx=8, n=3, f=8, out=PTR, ldo=8, drop=DropoutOpts(0.5, PTR, 0)) | args
    assert _lib.lib().rof_dropout(a["x"], a["t"], a["ldx"], a["n"], a["f"], a["out"], a["ldo"],
                                  None if a.get("no") else C.byref(a["drop"]), None) == code


@pytest.mark.parametrize("state,calls,used", [(None, 1, PTR), (PTR, 1, None), (PTR, -1, PTR + 16), (PTR, 1, PTR),
                                              (PTR + 4, 1, PTR + 16), (PTR, 1, PTR + 4), (PTR, 1, PTR + 8), (PTR + 8, 1, PTR)])
def test_dropout_state_refuses_what_it_cannot_run(state, calls, used):
    assert _lib.lib().rof_dropout_state_next(state, calls, used, None) == ARG


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    x, rng = torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RofError, match="CUDA tensor"):
        row_ops.layer_norm(x)
    with pytest.raises(RofError, match="CUDA tensor"):
        row_ops.dropout(x, 0.5, rng)
    with pytest.raises(RofError, match="on the GPU"):
        row_ops.ROF_DropoutState(3).next()
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(RofError, match="rate"):
            row_ops.ROF_Dropout(bad)
        with pytest.raises(RofError, match="rate"):
            row_ops.ROF_LayerNorm(4, dropout=bad)


def test_modules_hold_float32_parameters_and_the_generators_state():
    m = row_ops.ROF_LayerNorm(5)
    assert torch.equal(m.weight, torch.ones(5)) and torch.equal(m.bias, torch.zeros(5))
    assert set(m.state_dict()) == {"weight", "bias"}
    assert set(row_ops.ROF_LayerNorm(5, bias=False).state_dict()) == {"weight"}
    assert not row_ops.ROF_LayerNorm(5, elementwise_affine=False).state_dict()
    s = row_ops.ROF_DropoutState(11)
    assert s.state_dict()["state"].tolist() == [11, 0] and not list(s.parameters())
    x = torch.zeros(2, 3)
    assert row_ops.ROF_Dropout(0.5).eval()(x, None) is x and row_ops.ROF_Dropout(0.0)(x, None) is x


def test_models_take_norm_and_seed():
    from artifact_amd.ROF_models import ROF_GCN, ROF_GIN

    plain = ROF_GCN(6, 8, 3, 2, torch.relu, 0.5, reuse_size=0)
    assert not any(k.startswith(("norms", "dropout")) for k in plain.state_dict())
    for model in (ROF_GCN(6, 8, 3, 2, torch.relu, 0.5, norm="layer", dropout_seed=4),
                  ROF_GIN(6, 8, 3, 3, dropout=0.5, norm="layer", dropout_seed=4)):
        keys = {k for k in model.state_dict() if k.startswith(("norms", "dropout"))}
        assert keys == {"norms.0.weight", "norms.0.bias", "norms.1.weight", "norms.1.bias", "dropout_state.state"}
        assert isinstance(model.dropout, row_ops.ROF_Dropout) and model.dropout_state.state.tolist() == [4, 0]
    for bad in ("batch", True, 0):
        with pytest.raises(ValueError, match="norm"):
            ROF_GCN(6, 8, 3, 2, torch.relu, 0.5, norm=bad)
        with pytest.raises(ValueError, match="norm"):
            ROF_GIN(6, 8, 3, 3, norm=bad)
    with pytest.raises(RofError, match="rate"):
        ROF_GCN(6, 8, 3, 2, torch.relu, 1.5, dropout_seed=4)
