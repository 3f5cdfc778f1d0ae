"""How the row operators are called on the GPU: recorded programs, other streams, wrapped tensors."""
import ctypes as C
import io

import pytest
import torch
import torch.utils.checkpoint
from torch.fx.experimental.proxy_tensor import make_fx

from artifact_amd import _lib
from artifact_amd._lib import DropoutOpts, RofError
from artifact_amd.ROF_models import ROF_GCN
from artifact_amd.graphgen import features, make_workload
from artifact_amd.reuse_conv import build_input_info
from artifact_amd.row_ops import ROF_DropoutState, ROF_LayerNorm, dropout, layer_norm

pytestmark = pytest.mark.gpu


def rows(n, f, seed, dtype=torch.float32):
    return torch.randn(n, f, generator=torch.Generator().manual_seed(seed)).to("cuda", dtype)


def params(f, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1 + 0.3 * torch.randn(f, generator=gen)).cuda().requires_grad_(True),
            (0.3 * torch.randn(f, generator=gen)).cuda().requires_grad_(True))


def rng_tensor(seed=5, offset=3):
    return torch.tensor([seed, offset], device="cuda")


def model_on_a_graph(activation=torch.relu, **kw):
    ip, ix = make_workload("c1", 5)
    info = build_input_info(ip, ix, 3, device="cuda", min_consumers=2)
    torch.manual_seed(5)
    model = ROF_GCN(24, 20, 5, 2, activation, 0.4, reuse_size=info.reuse_size, kernel_type="ROF_v2", **kw).cuda()
    return model, info, torch.from_numpy(features(len(ip) - 1, 24, seed=1)).cuda()


def through_a_file(traced):
    buf = io.BytesIO()
    torch.jit.save(traced, buf)
    return torch.jit.load(io.BytesIO(buf.getvalue()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_traced_function_computes_what_it_traced(dtype):
    (w, b), rng = (t.detach() for t in params(24, 1)), rng_tensor()     # the tracer takes no leaves as constants
    calls = [lambda x: layer_norm(x, w, b), lambda x: layer_norm(x, w, b, relu=True, out_dtype=torch.bfloat16),
             lambda x: layer_norm(x, None, b, relu=True, dropout=0.5, rng=rng, call=2), lambda x: dropout(x, 0.25, rng, call=1),
             lambda x: dropout(layer_norm(x), 0.5, rng) * 2]
    with torch.no_grad():
        for call in calls:
            traced = torch.jit.trace(call, (rows(7, 24, 2, dtype),))
            assert "rof::" in str(traced.graph)
            for n in (7, 13, 1):
                x = rows(n, 24, 10 + n, dtype)
                assert torch.equal(traced(x), call(x)) and torch.equal(through_a_file(traced)(x), call(x))


def test_a_traced_program_checks_what_it_is_given():
    w, b = (t.detach() for t in params(24, 1))
    with torch.no_grad():
        traced = torch.jit.trace(lambda x: layer_norm(x, w, b), (rows(7, 24, 2),))
        for bad in (rows(7, 23, 3), rows(7, 24, 3).half(), rows(7, 24, 3).cpu(), rows(24, 7, 3).t()):
            with pytest.raises(RuntimeError):
                traced(bad)


class Tail(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = ROF_LayerNorm(24, relu=True, dropout=0.5)
        self.state = ROF_DropoutState(3)

    def forward(self, x):
        return self.norm(x, self.state.next(2), call=1)


def test_a_traced_module_draws_new_masks():
    m, other = Tail().cuda(), Tail().cuda()
    x = rows(40, 24, 2)
    with torch.no_grad():
        traced = torch.jit.trace(m, (x,), check_trace=False)     # a check would compare two masks
        m.state.state.copy_(torch.tensor([3, 0]))
        for _ in range(3):
            assert torch.equal(traced(x), other(x))
        assert m.state.state.tolist() == other.state.state.tolist() == [3, 6]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_recorded_step_computes_its_gradients(dtype):
    rng = rng_tensor()

    def step(x, w, b, dy):
        y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng)
        z = dropout(y, 0.25, rng, call=1)
        return (z.detach(),) + torch.autograd.grad(z, (x, w, b), dy)

    def inputs(n, seed):
        return (rows(n, 24, seed, dtype).requires_grad_(True), *params(24, seed + 1), rows(n, 24, seed + 2, dtype))

    recorded = make_fx(step)(*inputs(7, 1))
    targets = {str(node.target) for node in recorded.graph.nodes}
    assert {"rof.layer_norm.default", "rof.layer_norm_backward.default", "rof.dropout.default"} <= targets
    for seed in (20, 30):
        given = inputs(7, seed)
        assert all(torch.equal(s, t) for s, t in zip(recorded(*given), step(*given)))


def test_a_traced_network_computes_what_it_traced():
    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.first, self.norm, self.last = torch.nn.Linear(24, 20), ROF_LayerNorm(20, relu=True, dropout=0.4), torch.nn.Linear(20, 5)

        def forward(self, x):
            return self.last(self.norm(self.first(x)))

    net = Net().cuda().eval()
    with torch.no_grad():
        traced = through_a_file(torch.jit.trace(net, (rows(7, 24, 1),)))
        assert torch.equal(traced(rows(9, 24, 2)), net(rows(9, 24, 2)))


def test_torch_funcs_transforms_are_refused():
    x, (w, b), rng = rows(6, 8, 1), params(8, 2), rng_tensor()
    calls = [lambda x, w, b: layer_norm(x, w, b), lambda x, w, b: layer_norm(x, w, b, dropout=0.5, rng=rng)]
    for call in calls:
        for i in range(3):
            with pytest.raises(RofError, match="transforms"):
                torch.func.grad(lambda *t: call(*t).sum(), argnums=i)(x, w.detach(), b.detach())
        with pytest.raises(RofError, match="transforms"):
            torch.vmap(lambda w: call(x, w, b))(w.detach()[None])
    with pytest.raises(RofError, match="transforms"):
        torch.vmap(lambda r: dropout(x, 0.5, r))(rng[None])
    with pytest.raises(RofError, match="transforms"):
        torch.vmap(lambda s: ROF_DropoutState.next(type("S", (), {"state": s})()))(rng[None])


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("norm", ["layer", None])
def test_a_checkpointed_model_that_would_draw_other_masks_is_refused(norm, reentrant):
    model, info, x = model_on_a_graph(norm=norm, dropout_seed=3)
    x.requires_grad_(True)
    y = torch.utils.checkpoint.checkpoint(model, x, info, use_reentrant=reentrant)
    with pytest.raises(RofError, match="backward pass"):
        y.sum().backward()
    model.eval()                                             # no masks, no matter
    y = torch.utils.checkpoint.checkpoint(model, x, info, use_reentrant=reentrant)
    got, = torch.autograd.grad(model(x, info).sum(), x)
    x.grad = None
    y.sum().backward()
    assert torch.equal(x.grad, got)


def test_a_checkpointed_traced_module_that_would_draw_other_masks_is_refused():
    x = rows(9, 24, 1).requires_grad_(True)
    with torch.no_grad():
        traced = torch.jit.trace(Tail().cuda(), (x.detach(),), check_trace=False)
    y = torch.utils.checkpoint.checkpoint(traced, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="backward pass"):
        y.sum().backward()


@pytest.mark.parametrize("activation", [torch.relu, torch.tanh])
def test_the_models_call_their_norms(activation):
    """Hooks, pre-hooks and wrappers of a norm take part, and what they change is what the model computes with."""
    model, info, x = model_on_a_graph(norm="layer", dropout_seed=3, activation=activation)
    want, seen = model(x, info), []
    model.dropout_state.state.copy_(torch.tensor([3, 0]))
    handles = [n.register_forward_hook(lambda m, args, out: seen.append(out.shape)) for n in model.norms]
    assert torch.equal(model(x, info), want) and seen == [(len(x), 20)] * 2
    for h in handles:
        h.remove()
    weight = torch.linspace(0.5, 1.5, 20, device="cuda")

    def gather(m, args):
        m.weight.data.copy_(weight)

    model.norms[0].register_forward_pre_hook(gather)
    model.dropout_state.state.copy_(torch.tensor([3, 0]))
    got = model(x, info)
    assert not torch.equal(got, want)
    model.dropout_state.state.copy_(torch.tensor([3, 0]))
    other, _, _ = model_on_a_graph(norm="layer", dropout_seed=3, activation=activation)
    other.norms[0].weight.data.copy_(weight)
    assert torch.equal(other(x, info), got)
    torch.nn.utils.parametrizations.weight_norm(model.norms[1], dim=None)
    model(x, info).sum().backward()
    assert model.norms[1].parametrizations.weight.original0.grad is not None


def test_the_models_call_a_dropout_with_hooks():
    model, info, x = model_on_a_graph(norm="layer", dropout_seed=3)
    want, seen = model(x, info), []
    model.dropout_state.state.copy_(torch.tensor([3, 0]))
    model.dropout.register_forward_hook(lambda m, args, out: seen.append((args[0], out)))
    got = model(x, info)
    assert len(seen) == 2 and model.dropout_state.state.tolist() == [3, 2]
    rng = rng_tensor(3, 0)
    for i, (given, out) in enumerate(seen):
        assert torch.equal(out, dropout(given, 0.4, rng, call=i))
    # The same masks and sums, but the scale behind the norm's rounding, not in its parameters: 5 roundings of 2^-24 of values
    # up to 2 (3 + 0.3), which the next layer's 20 products and its norm (up to 4) magnify less than 100 times: below 2e-4
    assert torch.allclose(got, want, rtol=0, atol=2e-4)


def test_a_models_norm_with_a_relu_or_a_dropout_of_its_own():
    model, info, x = model_on_a_graph(norm="layer", dropout_seed=3, activation=torch.tanh)
    model.norms[0].relu, model.norms[1].p = True, 0.25
    got = model(x, info)
    assert model.dropout_state.state.tolist() == [3, 4]
    rng, h = rng_tensor(3, 0), x
    for i, (layer, norm) in enumerate(zip(model.layers, model.norms)):
        h = layer_norm(layer(h, info), norm.weight, norm.bias, relu=i == 0, dropout=0.25 if i else 0.0, rng=rng, call=2 + i)
        h = dropout(torch.tanh(h), 0.4, rng, call=i)
    assert torch.equal(model.layers[2](h, info), got)


def test_a_generator_state_with_the_negative_bit_is_refused():
    x, rng = rows(6, 8, 1), rng_tensor()
    state = ROF_DropoutState(3).cuda()
    state.state = state.state._neg_view()
    for call in (lambda: dropout(x, 0.5, rng._neg_view()), lambda: layer_norm(x, dropout=0.5, rng=rng._neg_view()), state.next):
        with pytest.raises(RofError, match="contiguous int64"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f", [3, 7, 47, 100, 256, 700, 1500, 4099, 7001])
def test_columns_without_a_weight_pass_the_gate_by_their_biass_sign(f, dtype):
    """Also where it is as small as numbers get, or zero, in the last column too; the others pass as ever."""
    n = 37
    x, (w, b), dy = rows(n, f, 1, dtype), params(f, 2), torch.ones(n, f, device="cuda")
    signs = torch.tensor([0.0, -0.0, 1e-40, -1e-40, 1e-9, -1e-9, 2.0, -2.0], device="cuda")
    at = torch.arange(f - 1, -1, -max(1, f // 8), device="cuda")[:8]
    for zero in (0.0, -0.0):
        with torch.no_grad():
            w[at], b[at] = zero, signs[:len(at)]
        h = x.double() - x.double().mean(1, keepdim=True)
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
        gate = h * w.detach().double() + b.detach().double() > 0
        db, = torch.autograd.grad(layer_norm(x, w, b, relu=True, out_dtype=torch.float32), b, dy)
        assert torch.equal(db.double(), gate.double().sum(0))       # whole numbers; every sign is settled in 64 bits
        assert torch.equal(db[at] > 0, signs[:len(at)] > 0)


def test_calls_on_a_busy_stream_wait_for_what_is_before_them():
    """Everything is on the device beforehand, so that nothing on the host waits for the stream: a kernel on any other stream
    would read the rows that the copy at the end of the queue is about to replace."""
    side = torch.cuda.Stream()
    w, b = params(64, 2)
    old, new, dy, rng = rows(50, 64, 1), rows(50, 64, 2), rows(50, 64, 3), rng_tensor()
    big = torch.randn(4096, 4096, device="cuda")
    state = ROF_DropoutState(8).cuda()

    def calls(x):
        used = state.next(2)
        y = layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng)
        return (y.detach(), used, dropout(x.detach(), 0.5, used)) + torch.autograd.grad(y, (x, w, b), dy)

    calls(old.clone().requires_grad_(True))              # kernels loaded, streams made
    want = calls(new.clone().requires_grad_(True))
    state.state.fill_(0)
    x, at = old.clone().requires_grad_(True), torch.tensor([8, 2], device="cuda")
    with torch.cuda.stream(side):
        big @ big
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(60):
            out = big @ big                              # tens of milliseconds
        x.detach().copy_(new)
        state.state.copy_(at)
        got = calls(x)
        busy = not side.query()
    torch.cuda.synchronize()
    assert busy and out.shape == big.shape
    assert all(torch.equal(s, t) for s, t in zip(got, want))


@pytest.mark.parametrize("dtype,f,n", [(torch.bfloat16, 512, 399996), (torch.bfloat16, 512, 399997), (torch.float32, 512, 399997),
                                       (torch.float32, 256, 399996), (torch.float32, 256, 399997), (torch.bfloat16, 16, 100000),
                                       (torch.float32, 5, 12799872), (torch.float32, 5, 12799873), (torch.bfloat16, 5, 12799873)])
def test_the_backward_launch_stays_in_its_workspace(dtype, f, n):
    L, st, kind = _lib.lib(), torch.cuda.current_stream().cuda_stream, 0 if dtype == torch.float32 else 1
    x = torch.randn(n, f, device="cuda", dtype=dtype)
    dy, (w, b), rng = x.flip(0), params(f, 2), rng_tensor()
    dx, dw, db = torch.empty_like(x), torch.empty(f, device="cuda"), torch.empty(f, device="cuda")
    size = L.rof_layer_norm_backward_workspace_bytes(n, f)
    ws = torch.full((size // 4 + 4096,), -7.0, device="cuda")
    opts = C.byref(DropoutOpts(0.5, rng.data_ptr(), 0))
    assert L.rof_layer_norm_backward(dy.data_ptr(), kind, f, x.data_ptr(), kind, f, n, f, w.data_ptr(), b.data_ptr(), 1e-5, 1, opts,
                                     dx.data_ptr(), f, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), size, st) == 0
    assert (ws[size // 4:] == -7).all()
    xx = x.requires_grad_(True)
    want = torch.autograd.grad(layer_norm(xx, w, b, relu=True, dropout=0.5, rng=rng), (xx, w, b), dy)
    assert all(torch.equal(s, t) for s, t in zip((dx, dw, db), want))


def test_a_traced_function_is_differentiable():
    (w, b), rng = (t.detach() for t in params(24, 1)), rng_tensor()

    def call(x):
        return dropout(layer_norm(x, w, b, relu=True), 0.5, rng)

    with torch.no_grad():
        traced = torch.jit.trace(call, (rows(7, 24, 2),))
    for n in (7, 11, 11, 11):                            # the interpreter specialises after its first runs
        x, dy = rows(n, 24, n).requires_grad_(True), rows(n, 24, 5)
        want, = torch.autograd.grad(call(x), x, dy)
        assert torch.equal(torch.autograd.grad(traced(x), x, dy)[0], want)


def test_a_batch_of_gradients_at_once():
    """is_grads_batched, which jacobian(vectorize=True) uses: one call of the operator for each."""
    x, (w, b), rng = rows(6, 8, 1).requires_grad_(True), params(8, 2), rng_tensor()
    batch = torch.stack([rows(6, 8, s) for s in (3, 4, 5)])
    for y, leaves in ((layer_norm(x, w, b, relu=True, dropout=0.5, rng=rng), (x, w, b)), (layer_norm(x, w, b), (w,)),
                      (dropout(x, 0.5, rng), (x,))):
        got = torch.autograd.grad(y, leaves, batch, is_grads_batched=True, retain_graph=True)
        for i, dy in enumerate(batch):
            want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            assert all(torch.equal(s[i], t) for s, t in zip(got, want))


@pytest.mark.parametrize("n,step,tol", [(16384, 64, 1.0), (6400000, 256, 3.0)])
def test_the_sums_over_workgroups_keep_small_terms_beside_a_large_one(n, step, tol):
    """One row of 2^24 and ones, `step` rows apart, which is what a workgroup takes at a time: added up in 32 bits a one would be
    lost beside 2^24.  In 64 bits what is left is half a step of 2^24, that is 1, for each time that a sum is stored: once, and
    in a workgroup and a chunk of workgroups before that where the launch is tiles."""
    x, (w, b) = rows(n, 16, 1), params(16, 2)
    dy = torch.zeros(n, 16, device="cuda")
    dy[::step] = 1.0
    dy[0] = 2.0 ** 24
    db, = torch.autograd.grad(layer_norm(x, w, b), b, dy)
    assert (db.double() - (2.0 ** 24 + n // step - 1)).abs().max().item() <= tol


def test_a_mode_that_answers_for_the_operators():
    """A dispatch mode may return what it likes without running them, also for arguments that they would refuse."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Answers(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return torch.empty_like(args[0]) if func is torch.ops.rof.dropout.default else func(*args, **(kwargs or {}))

    x = rows(6, 8, 1).requires_grad_(True)
    with Answers():
        y = dropout(x, 0.5, None)
    assert y.grad_fn is not None
    with pytest.raises(RuntimeError, match="rng"):
        y.sum().backward()


def test_export_and_compile():
    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = ROF_LayerNorm(24, relu=True)

        def forward(self, x):
            return self.norm(x * 2) + 1

    net, x, dy = Net().cuda(), rows(6, 24, 1).requires_grad_(True), rows(6, 24, 2)
    with pytest.raises(Exception, match="layer_norm"):
        torch.export.export(net, (x.detach(),))
    fast = torch.compile(net, backend="aot_eager")
    assert torch.equal(fast(x), net(x))
    assert torch.equal(torch.autograd.grad(fast(x), x, dy)[0], torch.autograd.grad(net(x), x, dy)[0])
