"""Row operators (artifact_amd.row_ops) on the GPU against their plain 64-bit forms, with the tolerances that row_oracle
derives from the roundings that 32 bits and the output's type allow."""
import ctypes as C

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from artifact_amd import _lib, row_ops
from artifact_amd._lib import DropoutOpts, RofError
from artifact_amd.row_ops import ROF_Dropout, ROF_DropoutState, ROF_LayerNorm, dropout, layer_norm
from row_oracle import HALF_STEP, U, Norm, kept, philox, scale, threshold

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
SEED, OFFSET = 0x1234567890ABCDEF, (1 << 33) + 5


def rows_of(n, f, dtype, seed, pitch=None, shift=0, mean=0.3):
    """n rows of f normally distributed columns, `pitch` elements apart and starting `shift` elements into their buffer."""
    pitch = pitch or f
    gen = torch.Generator().manual_seed(seed)
    data = torch.randn(n, f, generator=gen) * torch.exp(0.5 * torch.randn(n, 1, generator=gen)) + mean
    buf = torch.empty(n * pitch + shift, dtype=TYPES[dtype], device="cuda")
    t = buf.as_strided((n, f), (pitch, 1), shift)
    t.copy_(data)
    return t


def params(f, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1 + 0.3 * torch.randn(f, generator=gen)).cuda().requires_grad_(True),
            (0.3 * torch.randn(f, generator=gen)).cuda().requires_grad_(True))


def rng_tensor(seed=SEED, offset=OFFSET):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def host(t):
    return t.detach().double().cpu().numpy()


def near(got, want, tol, what):
    """Within tol, plus half a step of the type it is stored in (of the value as computed, tol included)."""
    g = host(got)
    tol = tol + HALF_STEP[str(got.dtype).replace("torch.", "")] * (np.abs(want) + tol)
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(g - want) / np.maximum(tol, 1e-300)):.3f} "
                           f"of the tolerance, first at {np.argwhere(bad)[0]}")


def check_norm(x, w, b, dy, relu=False, p=0.0, call=0, out_dtype=None, eps=1e-5):
    rng = rng_tensor() if p else None
    x = x.detach().requires_grad_(True)
    y = layer_norm(x, w, b, eps=eps, relu=relu, dropout=p, rng=rng, call=call, out_dtype=out_dtype)
    keep = kept(np.arange(x.shape[0]), x.shape[1], p, SEED, OFFSET + call) if p else None
    o = Norm(host(x), None if w is None else host(w), None if b is None else host(b), eps, relu, keep, p)
    assert y.dtype == (out_dtype or x.dtype) and y.is_contiguous()
    near(y, o.y, o.y_tol, "y")
    if p:
        assert not host(y)[~keep].any()
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    want, tol = o.backward(host(dy))
    names = ["dx"] + (["dweight"] if w is not None else []) + (["dbias"] if b is not None else [])
    pick = {"dx": 0, "dweight": 1, "dbias": 2}
    for name, g in zip(names, grads):
        near(g, want[pick[name]], tol[pick[name]], name)
    return (y,) + grads


# a row per lane group, per wavefront, per four and per sixteen of them, each at its borders; odd numbers of rows and columns
SHAPES = [(1, 1), (3, 2), (2, 3), (5, 4), (64, 5), (130, 8), (7, 9), (33, 15), (257, 16), (19, 17), (65, 31), (16, 32), (70, 33),
          (50, 47), (21, 63), (100, 64), (35, 65), (33, 100), (41, 127), (18, 128), (11, 129), (64, 255), (40, 256), (17, 257),
          (9, 511), (7, 513), (6, 1000), (9, 1024), (6, 1025), (5, 2047), (5, 2048), (6, 2049), (4, 4096), (4, 4097), (3, 4608), (3, 4609), (3, 8191),
          (2, 8192), (3, 6145), (9, 1537), (9, 1536), (9, 2304), (9, 2305)]
WIDE = [(2, 8193), (3, 12289), (2, 16384)]          # bfloat16 only: rows of at most 32 KB


@pytest.mark.parametrize("xt,yt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n,f", SHAPES)
def test_layer_norm_and_its_gradient(n, f, xt, yt):
    w, b = params(f, f)
    check_norm(rows_of(n, f, xt, n + f), w, b, rows_of(n, f, yt, n + f + 1), out_dtype=TYPES[yt])


@pytest.mark.parametrize("xt,yt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("n,f", SHAPES)
@pytest.mark.parametrize("relu,p", [(True, 0.5), (True, 0.0), (False, 0.3)])
def test_the_tail_of_a_hidden_layer_and_its_gradient(n, f, xt, yt, relu, p):
    w, b = params(f, f + 7)
    check_norm(rows_of(n, f, xt, n + f), w, b, rows_of(n, f, yt, n + f + 1), relu, p, call=3, out_dtype=TYPES[yt])


@pytest.mark.parametrize("yt", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,f", WIDE)
@pytest.mark.parametrize("relu,p", [(False, 0.0), (True, 0.5)])
def test_the_widest_rows(n, f, yt, relu, p):
    w, b = params(f, f)
    check_norm(rows_of(n, f, "bfloat16", n + f), w, b, rows_of(n, f, yt, n + f + 1), relu, p, out_dtype=TYPES[yt])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,f", [(20000, 16), (5001, 47), (3000, 256), (70001, 100)])
def test_more_rows_than_one_launch_holds_at_a_time(n, f, dtype):
    w, b = params(f, 3)
    check_norm(rows_of(n, f, dtype, 5), w, b, rows_of(n, f, dtype, 6), True, 0.5)


@pytest.mark.parametrize("dtype,n,f", [("float32", (1 << 18) + 3, 200), ("bfloat16", (1 << 18) + 77, 500), ("float32", (1 << 20) + 5, 33),
                                       ("float32", (1 << 24) + 3, 3), ("bfloat16", (1 << 24) + 259, 5), ("float32", (1 << 23) + 1, 7),
                                       ("float32", 400001, 200), ("float32", 399996, 256), ("float32", 399997, 200), ("bfloat16", 400033, 500),
                                       ("float32", 3200001, 47), ("bfloat16", 1600019, 300), ("float32", 800005, 150),
                                       ("float32", 25600003, 3), ("bfloat16", 12800077, 13)])
def test_parameter_gradients_of_matrices_in_tiles(dtype, n, f):
    """So many rows that the backward launch leaves thousands of partial rows, which two more launches add up.  The 64-bit
    form is evaluated on the GPU here; the tolerances are row_oracle's."""
    x, dy = rows_of(n, f, dtype, 1, mean=0.0).requires_grad_(True), rows_of(n, f, dtype, 2)
    w, b = params(f, 3)
    dx, dw, db = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    x64, d = x.detach().double(), dy.double()
    m = x64.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x64 - m) ** 2).mean(1, keepdim=True) + 1e-5)
    h, a = (x64 - m) * r, 128 * U * (r * (x64.abs() + m.abs()) + 1)
    adds = -(-n // 1024) + 104
    near(dw, host((d * h).sum(0)), host((d.abs() * a).sum(0) + adds * U * (d * h).abs().sum(0)), "dweight")
    near(db, host(d.sum(0)), host(adds * U * d.abs().sum(0)), "dbias")
    rows = [0, 1, n // 2, n - 2, n - 1]
    o = Norm(host(x[rows]), host(w), host(b))
    want, tol = o.backward(host(dy[rows]))
    near(dx[rows], want[0], tol[0], "dx")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("f,pitch,shift", [(47, 48, 0), (47, 49, 1), (64, 72, 0), (64, 65, 3), (100, 104, 1), (1025, 1027, 1),
                                           (4097, 4100, 1), (256, 1000, 5)])
def test_rows_apart_and_off_the_vectors_boundaries(f, pitch, shift, dtype):
    w, b = params(f, 1)
    a = check_norm(rows_of(37, f, dtype, 2, pitch, shift), w, b, rows_of(37, f, dtype, 3, pitch + 1, shift + 1), True, 0.4)
    c = check_norm(rows_of(37, f, dtype, 2), w, b, rows_of(37, f, dtype, 3), True, 0.4)
    assert all(torch.equal(s, t) for s, t in zip(a, c))       # the strides change no bit


@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("f", [47, 256, 1500])
def test_parameters_may_be_left_out(f, with_w, with_b):
    w, b = params(f, 1)
    check_norm(rows_of(29, f, "float32", 2), w if with_w else None, b if with_b else None, rows_of(29, f, "float32", 3), True, 0.2)


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
def test_only_the_gradients_that_are_wanted(wanted):
    x, (w, b) = rows_of(300, 40, "float32", 1), params(40, 2)
    dy = rows_of(300, 40, "float32", 3)
    full = check_norm(x, w, b, dy, True)[1:]
    leaves = [t.detach().requires_grad_(bool(i)) for t, i in zip((x, w, b), wanted)]
    y = layer_norm(*leaves, relu=True)
    got = torch.autograd.grad(y, [t for t, i in zip(leaves, wanted) if i], dy)
    assert all(torch.equal(g, t) for g, t in zip(got, [t for t, i in zip(full, wanted) if i]))


def test_no_rows():
    w, b = params(12, 1)
    x = torch.empty(0, 12, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng_tensor())
    assert y.shape == (0, 12)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 12, device="cuda"))
    assert dx.shape == (0, 12) and not dw.any() and not db.any()
    assert dropout(x, 0.5, rng_tensor()).shape == (0, 12)


@pytest.mark.parametrize("f", [1, 16, 47, 1030])
def test_rows_without_spread(f):
    """A constant row has variance 0: h = 0 exactly where the mean is exact, dx is r (g - mean g) with r = eps^-1/2."""
    x = torch.tensor([0.0, 1.0, -8.0, 0.0], device="cuda")[:, None].expand(4, f).contiguous()
    w, b = params(f, 2)
    y = check_norm(x, w, b, rows_of(4, f, "float32", 3), True)[0]
    assert torch.equal(y, torch.relu(b.detach()).expand(4, f))


@pytest.mark.parametrize("f", [16, 47, 256, 1500, 5000])
@pytest.mark.parametrize("mean", [30.0, 300.0])
def test_rows_far_from_zero(f, mean):
    w, b = params(f, 4)
    check_norm(rows_of(40, f, "float32", 5, mean=mean), w, b, rows_of(40, f, "float32", 6), True, 0.5)


@pytest.mark.parametrize("f", [7, 47, 300, 1500, 6000])
def test_a_row_with_infinity_or_nan_spoils_no_other(f):
    x = rows_of(9, f, "float32", 1)
    w, b = params(f, 2)
    dy = rows_of(9, f, "float32", 3)
    clean = check_norm(x, w, b, dy, True, 0.3)
    y0, dx0 = clean[0].clone(), clean[1].clone()
    x[2, f // 2], x[5, 0], x[7, f - 1] = float("inf"), float("nan"), -float("inf")
    x.requires_grad_(True)
    y = layer_norm(x, w, b, relu=True, dropout=0.3, rng=rng_tensor())
    dx, = torch.autograd.grad(y, x, dy)
    keep = torch.from_numpy(kept(np.arange(9), f, 0.3, SEED, OFFSET)).cuda()
    others = [0, 1, 3, 4, 6, 8]
    assert torch.equal(y[others], y0[others]) and torch.equal(dx[others], dx0[others])
    for r in (2, 5, 7):
        assert torch.isnan(y[r][keep[r]]).all() and not y[r][~keep[r]].any()    # a dropped element is 0 whatever it was


def test_the_relus_gate_is_the_sign_of_the_exact_value():
    """Biases that cancel h w to the last bit of float32 in one column after the other: a gate decided in 32 bits would be a
    coin toss there, and its error a whole gradient."""
    for f in (16, 47, 256, 1500, 5000):
        n = 64
        x, (w, _) = rows_of(n, f, "float32", f), params(f, 2)
        o = Norm(host(x), host(w))
        at = np.arange(f) % n
        b = torch.from_numpy(-(o.h * o.w)[at, np.arange(f)].astype(np.float32)).cuda()
        o = Norm(host(x), host(w), host(b), relu=True)
        assert np.median(np.abs(o.pre[at, np.arange(f)])) < 1e-7 and (np.abs(o.pre[at, np.arange(f)]) > 1e-13).mean() > 0.99
        x.requires_grad_(True)
        dy = torch.ones(n, f, device="cuda")
        db_want = o.gate.sum(0)
        bias = b.requires_grad_(True)
        db, = torch.autograd.grad(layer_norm(x, w, bias, relu=True), bias, dy)
        sure = (np.abs(o.pre) > 1e-13).all(0)
        assert np.array_equal(host(db)[sure], db_want[sure])       # small whole numbers: exact in float32


@pytest.mark.parametrize("relu,p", [(False, 0.0), (False, 0.4)])
def test_the_gradient_is_the_difference_quotient(relu, p):
    """Along a direction: the kernel's own values at both ends against its gradient.  The values are off by y_tol each, which
    the quotient divides by the step; its curvature is taken from the 64-bit form at the same points."""
    n, f, step = 23, 47, 2.0 ** -6
    x, (w, b) = rows_of(n, f, "float32", 1), params(f, 2)
    dy, v = rows_of(n, f, "float32", 3), rows_of(n, f, "float32", 4)
    keep = kept(np.arange(n), f, p, SEED, OFFSET) if p else None
    ends, exact, tol = [], [], 0.0
    for s in (step, -step):
        t = (x + s * v).detach()
        y = layer_norm(t, w, b, dropout=p, rng=rng_tensor() if p else None)
        o = Norm(host(t), host(w), host(b), keep=keep, p=p)
        ends.append((host(y) * host(dy)).sum())
        exact.append((o.y * host(dy)).sum())
        tol += ((o.y_tol + HALF_STEP["float32"] * np.abs(o.y)) * np.abs(host(dy))).sum() / (2 * step)
    o = Norm(host(x), host(w), host(b), keep=keep, p=p)
    want, gtol = o.backward(host(dy))
    curve = abs((exact[0] - exact[1]) / (2 * step) - (want[0] * host(v)).sum())
    xx = x.detach().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(xx, w, b, dropout=p, rng=rng_tensor() if p else None), xx, dy)
    along = (host(dx) * host(v)).sum()
    tol += ((gtol[0] + HALF_STEP["float32"] * np.abs(want[0])) * np.abs(host(v))).sum()
    # x +- step v is rounded to float32 once: half a step of it, through the gradient
    tol += (np.abs(want[0]) * HALF_STEP["float32"] * (np.abs(host(x)) + step * np.abs(host(v)))).sum() * 2 / (2 * step)
    assert abs((ends[0] - ends[1]) / (2 * step) - along) <= tol + curve


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,f,pitch,shift", [(1, 1, 1, 0), (1, 7, 7, 1), (3, 8, 8, 0), (1000, 16, 16, 0), (333, 47, 48, 0), (333, 47, 47, 1),
                                             (129, 100, 101, 3), (64, 256, 256, 0), (5, 4099, 4100, 1), (2, 70001, 70001, 0),
                                             (60001, 33, 33, 0), (20003, 256, 256, 0), (1 << 18, 8, 8, 0)])
@pytest.mark.parametrize("p", [0.5, 0.13])
def test_dropout_is_its_definition_to_the_bit(n, f, pitch, shift, dtype, p):
    x = rows_of(n, f, dtype, 1, pitch, shift).requires_grad_(True)
    dy = rows_of(n, f, dtype, 2, pitch + 1, shift)
    y = dropout(x, p, rng_tensor(), call=7)
    dx, = torch.autograd.grad(y, x, dy)
    keep = torch.from_numpy(kept(np.arange(n), f, p, SEED, OFFSET + 7)).cuda()
    for got, src in ((y, x.detach()), (dx, dy)):
        # one product in float32, rounded once to the type: what torch computes as well
        assert torch.equal(got, torch.where(keep, src.float() * np.float32(scale(p)), 0.0).to(src.dtype))
        assert got.is_contiguous()


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -17, 1.0 - 2.0 ** -18, 1.0])
def test_dropout_at_the_ends_of_the_range(p):
    x = rows_of(200, 47, "float32", 1)
    x[3, 4], x[5, 6] = float("nan"), float("inf")
    keep = torch.from_numpy(kept(np.arange(200), 47, p, SEED, OFFSET)).cuda()
    y = dropout(x, p, rng_tensor())
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(torch.where(keep, x * np.float32(scale(p)), 0.0)))
    assert torch.isfinite(y[~keep]).all()
    if p == 1.0:
        z = layer_norm(x, relu=True, dropout=1.0, rng=rng_tensor())
        assert not z.any()


def test_a_mask_depends_on_the_place_and_the_generator_alone():
    """Not on the type, the strides, or whether norm and dropout are one pass or two."""
    n, f = 77, 100
    ones = torch.ones(n, f, device="cuda")
    a = dropout(ones, 0.5, rng_tensor()) > 0
    assert torch.equal(a, dropout(ones.bfloat16(), 0.5, rng_tensor()) > 0)
    assert torch.equal(a, dropout(torch.ones(n, 130, device="cuda")[:, 3:103], 0.5, rng_tensor()) > 0)
    z = layer_norm(rows_of(n, f, "float32", 1), None, torch.full((f,), 100.0, device="cuda"), dropout=0.5, rng=rng_tensor())
    assert torch.equal(a, z > 0)
    assert not torch.equal(a, dropout(ones, 0.5, rng_tensor(), call=1) > 0)
    assert torch.equal(dropout(ones, 0.5, rng_tensor(), call=1), dropout(ones, 0.5, rng_tensor(offset=OFFSET + 1)))
    assert torch.equal(dropout(ones, 0.5, rng_tensor(-5, -1)) > 0, torch.from_numpy(kept(np.arange(n), f, 0.5, -5, -1)).cuda())


@pytest.mark.parametrize("dtype,f,n", [("bfloat16", 300, (1 << 23) + 5), ("float32", 513, (1 << 22) + 3)])
def test_rows_beyond_the_reach_of_32_bit_offsets(dtype, f, n):
    """More than 2^31 elements: the rows on both sides of every 2^31, 2^32 elements and bytes, and the last ones."""
    x = torch.empty(n, f, dtype=TYPES[dtype], device="cuda")
    size = x.element_size()
    rows = sorted({r for e in (1 << 31, 1 << 32) for u in (1, size) for r in (e // u // f - 1, e // u // f, e // u // f + 1)
                   if 0 <= r < n} | {0, n - 2, n - 1})
    for part in x.split(1 << 20):
        part.normal_()
    dy = x.flip(0)
    w, b = params(f, 2)
    y = dropout(x, 0.5, rng_tensor())
    keep = kept(np.array(rows), f, 0.5, SEED, OFFSET)
    assert np.array_equal(host(y[rows]), host(torch.where(torch.from_numpy(keep).cuda(), x[rows].float() * 2, 0.0).to(x.dtype)))
    del y
    x.requires_grad_(True)
    y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng_tensor())
    dx, = torch.autograd.grad(y, x, dy)
    o = Norm(host(x[rows]), host(w), host(b), relu=True, keep=keep, p=0.5)
    near(y[rows], o.y, o.y_tol, "y")
    want, tol = o.backward(host(dy[rows]))
    near(dx[rows], want[0], tol[0], "dx")


def test_the_c_abi_leaves_what_is_between_and_behind_the_rows():
    """Output rows apart: the columns between them and the rows behind the last one keep what they held."""
    L, n, f = _lib.lib(), 21, 47
    st = torch.cuda.current_stream().cuda_stream
    x, (w, b), rng = rows_of(n, f, "float32", 1), params(f, 2), rng_tensor()
    dy = rows_of(n, f, "float32", 3)
    opts = C.byref(DropoutOpts(0.5, rng.data_ptr(), 0))
    for ld in (48, 50, 64):
        y, dx, z = (torch.full((n + 3, ld), -7.0, device="cuda") for _ in range(3))
        dw, db = torch.empty(f, device="cuda"), torch.empty(f, device="cuda")
        size = L.rof_layer_norm_backward_workspace_bytes(n, f)
        ws = torch.full((size // 4 + 64,), -7.0, device="cuda")
        assert L.rof_layer_norm(x.data_ptr(), 0, f, n, f, w.data_ptr(), b.data_ptr(), 1e-5, 1, opts, y.data_ptr(), 0, ld, st) == 0
        assert L.rof_layer_norm_backward(dy.data_ptr(), 0, f, x.data_ptr(), 0, f, n, f, w.data_ptr(), b.data_ptr(), 1e-5, 1, opts,
                                         dx.data_ptr(), ld, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), size, st) == 0
        assert L.rof_dropout(x.data_ptr(), 0, f, n, f, z.data_ptr(), ld, opts, st) == 0
        xx = x.detach().requires_grad_(True)
        want = layer_norm(xx, w, b, relu=True, dropout=0.5, rng=rng)
        assert torch.equal(y[:n, :f], want) and torch.equal(z[:n, :f], dropout(x, 0.5, rng))
        for g, t in zip((dx[:n, :f], dw, db), torch.autograd.grad(want, (xx, w, b), dy)):
            assert torch.equal(g, t)
        for t in (y, dx, z):
            assert (t[n:] == -7).all() and (t[:, f:] == -7).all()
        assert (ws[size // 4:] == -7).all()


def test_repeated_calls_give_the_same_bits():
    x, (w, b) = rows_of(30000, 100, "float32", 1).requires_grad_(True), params(100, 2)
    dy = rows_of(30000, 100, "float32", 3)

    def once():
        y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng_tensor())
        return (y,) + torch.autograd.grad(y, (x, w, b), dy)

    first = once()
    for _ in range(3):
        assert all(torch.equal(s, t) for s, t in zip(first, once()))


def test_broadcast_and_transposed_gradients():
    x, (w, b) = rows_of(40, 24, "float32", 1).requires_grad_(True), params(24, 2)
    y = layer_norm(x, w, b)
    one = torch.ones((), device="cuda")
    for dy in (one.expand(40, 24), torch.ones(24, device="cuda").expand(40, 24), torch.ones(40, 1, device="cuda").expand(40, 24)):
        got = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
        want = torch.autograd.grad(y, (x, w, b), torch.ones(40, 24, device="cuda"), retain_graph=True)
        assert all(torch.equal(s, t) for s, t in zip(got, want))
    t = rows_of(24, 40, "float32", 5)
    got = torch.autograd.grad(y, (x, w, b), t.t(), retain_graph=True)
    want = torch.autograd.grad(y, (x, w, b), t.t().contiguous(), retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
    z = dropout(x, 0.5, rng_tensor())
    assert torch.equal(torch.autograd.grad(z.sum(), x)[0], dropout(torch.ones_like(x), 0.5, rng_tensor()))


def test_on_another_stream():
    side = torch.cuda.Stream()
    w, b = params(64, 2)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            big = big @ big * 1e-3          # work that the stream has to get through first
        x = rows_of(50, 64, "float32", 1)
        check_norm(x, w, b, rows_of(50, 64, "float32", 3), True, 0.5)
    side.synchronize()


def test_two_streams_at_once():
    w, b = params(256, 2)
    xs = [rows_of(20000, 256, "bfloat16", i).requires_grad_(True) for i in range(2)]
    dy = rows_of(20000, 256, "bfloat16", 9)

    def once(x):
        y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    rng = rng_tensor()
    want = [once(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = once(xs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for g, h in zip(got, want) for s, t in zip(g, h))


def test_the_state_moves_on_and_a_step_keeps_its_values():
    state = ROF_DropoutState(42).cuda()
    a, b = state.next(3), state.next()
    assert a.tolist() == [42, 0] and b.tolist() == [42, 3] and state.state.tolist() == [42, 4]
    other = ROF_DropoutState(0).cuda()
    other.load_state_dict(state.state_dict())
    assert other.next().tolist() == [42, 4]
    # the state itself as rng: moving it on before the backward pass would change the mask, and is an error
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    y = dropout(x, 0.5, state.state)
    state.next()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_a_captured_step_draws_new_masks_at_every_replay():
    n, f = 500, 64
    x, dy = rows_of(n, f, "float32", 1).requires_grad_(True), rows_of(n, f, "float32", 2)
    w, b = params(f, 3)
    state = ROF_DropoutState(9).cuda()

    def step(rng):
        y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng)
        z = dropout(y, 0.25, rng, call=1)
        return (z.detach(),) + torch.autograd.grad(z, (x, w, b), dy)    # no autograd graph outlives the step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state.next(2))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(state.next(2))
    at = int(state.state[1])
    masks = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step(torch.tensor([9, at + 2 * i], device="cuda"))
        assert all(torch.equal(s, t) for s, t in zip(got, want)), i
        masks.append(got[0] != 0)
        torch.cuda.synchronize()
    assert int(state.state[1]) == at + 8
    assert not torch.equal(masks[0], masks[1])


def test_two_captured_graphs_replayed_in_turn():
    cases = []
    for i in range(2):
        w, b = params(47, 3)       # leaves of its own: a capture and another live autograd graph must not share any
        x, dy = rows_of(3000, 47, "float32", i).requires_grad_(True), rows_of(3000, 47, "float32", 5 + i)
        rng = rng_tensor(i, i)

        def step(x=x, w=w, b=b, dy=dy, rng=rng):
            y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng)
            return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)   # no autograd graph outlives the step

        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        cases.append((graph, outs, want, step))      # step holds the inputs, which the graph reads
    for _ in range(3):
        for graph, _, _, _ in cases:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs, want, _ in cases:
            assert all(torch.equal(s, t) for s, t in zip(outs, want))


def test_refusals():
    x, rng = torch.randn(6, 8, device="cuda"), rng_tensor()
    w = torch.ones(8, device="cuda")
    for bad in (x.half(), x.double(), x[0], x.t(), x[:, :0], x[:1].expand(6, 8), x[:, ::2]):
        with pytest.raises(RofError):
            layer_norm(bad)
        with pytest.raises(RofError):
            dropout(bad, 0.5, rng)
    for bad in (w[:4], w.half(), w.cpu(), torch.ones(16, device="cuda")[::2], w[None]):
        with pytest.raises(RofError, match="weight"):
            layer_norm(x, bad)
        with pytest.raises(RofError, match="bias"):
            layer_norm(x, w, bad)
    for bad in (None, rng.cpu(), rng.int(), torch.zeros(3, dtype=torch.int64, device="cuda"),
                torch.zeros(4, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(RofError, match="rng"):
            dropout(x, 0.5, bad)
        with pytest.raises(RofError, match="rng"):
            layer_norm(x, dropout=0.5, rng=bad)
    for bad in (-0.5, 1.5, float("nan")):
        with pytest.raises(RofError, match="rate"):
            dropout(x, bad, rng)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(RofError, match="eps"):
            layer_norm(x, eps=bad)
    with pytest.raises(RofError, match="out_dtype"):
        layer_norm(x, out_dtype=torch.float16)
    for bad in (torch.zeros(1, 8193, device="cuda"), torch.zeros(1, 16385, dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(RofError, match="at most"):
            layer_norm(bad)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: layer_norm(dual), lambda: dropout(dual, 0.5, rng)):
            with pytest.raises(RofError, match="forward-mode"):
                call()
    y = layer_norm(x.requires_grad_(True))
    g, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):                              # no second derivative
        torch.autograd.grad(g.sum(), x)


def test_modules_follow_their_mode():
    x, rng = rows_of(30, 16, "float32", 1), rng_tensor()
    m = ROF_LayerNorm(16, relu=True, dropout=0.5).cuda()
    with torch.no_grad():
        assert torch.equal(m(x, rng), layer_norm(x, m.weight, m.bias, relu=True, dropout=0.5, rng=rng))
        m.eval()
        assert torch.equal(m(x), layer_norm(x, m.weight, m.bias, relu=True))
    d = ROF_Dropout(0.5)
    assert torch.equal(d(x, rng, 2), dropout(x, 0.5, rng, 2))
    assert d.eval()(x, None) is x


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("f", [2, 7, 47, 100, 300, 517, 1500, 4099, 6001])
@pytest.mark.parametrize("relu,p", [(True, 0.0), (False, 0.5), (True, 0.5)])
def test_a_gradient_that_is_masked_may_be_anything(f, dtype, bad, relu, p):
    """Where the ReLU or the dropout stops the gradient, infinity and NaN in it leave dx and the parameters' gradients as
    they were, in the last column too, whose vector also covers columns that the row does not have."""
    n = 13
    x, (w, b), dy = rows_of(n, f, dtype, 1), params(f, 2), rows_of(n, f, dtype, 3)
    want = check_norm(x, w, b, dy, relu, p)
    rows = np.arange(n)
    keep = kept(rows, f, p, SEED, OFFSET) if p else np.ones((n, f), dtype=bool)
    gone = ~keep | (relu & (Norm(host(x), host(w), host(b)).pre <= 0))
    assert gone[:, -1].any() and gone[:, :-1].any()
    dy[torch.from_numpy(gone).cuda()] = bad
    x = x.detach().requires_grad_(True)
    y = layer_norm(x, w, b, relu=relu, dropout=p, rng=rng_tensor())
    for got, t in zip(torch.autograd.grad(y, (x, w, b), dy), want[1:]):
        assert torch.equal(got, t)


def test_views_and_derivatives_that_are_refused():
    x, rng, w = torch.randn(6, 8, device="cuda"), rng_tensor(), torch.ones(8, device="cuda")
    dual_level, make_dual = torch.autograd.forward_ad.dual_level, torch.autograd.forward_ad.make_dual
    calls = [lambda t: layer_norm(t), lambda t: dropout(t, 0.5, rng)]
    for call in calls:
        with pytest.raises(RofError, match="negative"):
            call(x._neg_view())
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)
        with pytest.raises(RuntimeError):
            torch.vmap(call)(x[None])
        with dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            t = x.detach().requires_grad_(True)
            torch.autograd.grad(call(t), t, make_dual(x, x))
    with pytest.raises(RofError, match="weight"):
        layer_norm(x, w._neg_view())
    with dual_level():
        with pytest.raises(RofError, match="forward-mode"):
            layer_norm(x, make_dual(w, w))
        with pytest.raises(RofError, match="forward-mode"):
            layer_norm(x, w, make_dual(w, w))


def test_a_gradient_with_the_negative_bit():
    x, dy = rows_of(6, 8, "float32", 1).requires_grad_(True), rows_of(6, 8, "float32", 2)
    for call in (lambda: layer_norm(x), lambda: dropout(x, 0.5, rng_tensor())):
        assert torch.equal(torch.autograd.grad(call(), x, dy._neg_view())[0], torch.autograd.grad(call(), x, -dy)[0])


def test_what_the_backward_pass_keeps_is_watched_over():
    dy = rows_of(6, 8, "float32", 2)
    for which in range(3):
        x, (w, b) = rows_of(6, 8, "float32", 1).requires_grad_(True), params(8, 3)
        y = layer_norm(x, w, b, relu=True)
        with torch.no_grad():
            (x, w, b)[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, (x, w, b), dy)
    x, (w, b) = rows_of(6, 8, "float32", 1).requires_grad_(True), params(8, 3)
    for call in (lambda: layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng_tensor()), lambda: dropout(x, 0.5, rng_tensor())):
        y = call()
        want = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
        with pytest.raises(RuntimeError, match="a second time"):
            torch.autograd.grad(y, x, dy)
        with torch.autograd.graph.save_on_cpu():
            y = call()
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def test_a_checkpointed_part_draws_the_mask_of_its_first_pass():
    state, dy = ROF_DropoutState(3).cuda(), rows_of(40, 16, "float32", 2)
    x, (w, b) = rows_of(40, 16, "float32", 1).requires_grad_(True), params(16, 3)
    part = lambda x, rng: dropout(layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng), 0.3, rng, call=1) * 2   # noqa: E731
    rng = state.next(2)
    want = torch.autograd.grad(part(x, rng), (x, w, b), dy)
    y = torch.utils.checkpoint.checkpoint(part, x, rng, use_reentrant=False)
    state.next(2)
    assert all(torch.equal(g, t) for g, t in zip(torch.autograd.grad(y, (x, w, b), dy), want))


@pytest.mark.parametrize("dtype,mean", [("float32", 0.0), ("float32", 20.0), ("float32", 500.0), ("bfloat16", 20.0)])
@pytest.mark.parametrize("f", [5, 47, 150, 256, 700, 1500, 2700, 4099, 8000])
def test_the_relus_gate_in_rows_of_levels(f, dtype, mean):
    """As above, with rows whose parts have means of their own, on both sides of the row's and far from zero: the error of a
    wavefront's mean then counts in the row's spread as well."""
    n = 96
    level = torch.where(torch.arange(f) * 3 // f % 2 == 1, -1.0, 1.0) + mean
    x = rows_of(n, f, dtype, f, mean=0.0)
    x.copy_(0.05 * x.float() + level.cuda())
    w, _ = params(f, 2)
    o = Norm(host(x), host(w))
    at = np.arange(f) % n
    b = torch.from_numpy(-(o.h * o.w)[at, np.arange(f)].astype(np.float32)).cuda().requires_grad_(True)
    o = Norm(host(x), host(w), host(b), relu=True)
    db, = torch.autograd.grad(layer_norm(x, w, b, relu=True), b, torch.ones_like(x))
    sure = (np.abs(o.pre) > 1e-12 * (1 + mean)).all(0)         # beyond the rounding of 64 bits
    assert sure.mean() > 0.9
    assert np.array_equal(host(db)[sure], o.gate.sum(0)[sure])


@pytest.mark.parametrize("n,f", [(1, (1 << 31) - 1), (1, (1 << 31) - 8), (3, (1 << 30) + 5)])
def test_dropout_of_the_longest_rows(n, f):
    x = torch.full((n, f), 3.0, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.25, rng_tensor())
    groups = (f + 7) // 8
    for row in range(n):
        for first in (0, groups // 2 - 2, groups - 40):
            g = np.arange(first, min(first + 40, groups))
            i = g.astype(np.uint64) + np.uint64(row * groups)
            c = np.zeros((len(i), 4), dtype=np.uint64)
            c[:, 0], c[:, 1], c[:, 2], c[:, 3] = i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), OFFSET & 0xFFFFFFFF, OFFSET >> 32
            w = philox(c, (SEED & 0xFFFFFFFF, SEED >> 32))
            u = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(-1)
            got = host(y[row, 8 * first: 8 * first + len(u)])
            want = np.where(u >= threshold(0.25), host(torch.tensor(3 * scale(0.25), dtype=torch.float32).bfloat16()), 0.0)
            assert np.array_equal(got, want[:len(got)]) and len(got) >= len(u) - 7
