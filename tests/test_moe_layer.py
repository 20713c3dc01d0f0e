"""What the example layer keeps, for how long, and what autograd sees of it: its own
classes on the CPU, over operators that stand in for the kernels. Like the kernels
they write the caller's buffers behind autograd's back (`.data`: no version counts)."""
import gc
import weakref
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

import mini_triton_nvgpu_v1_amd as tb  # noqa: E402
from mini_triton_nvgpu_v1_amd import moe_layer  # noqa: E402


class _Desc:
    """Products grouped by expert, in 32 bits."""

    def __init__(self, log, fields):
        self.log = log
        self.f = {"kind": tb.GROUPED_ROWS, "b_layout": tb.B_KN, "activation": tb.ACT_NONE,
                  **fields}

    def launch(self, a, b, c, offsets=None, rows=None, a_scale=None, b_scale=None, **_):
        f = self.f
        self.log.append("wgrad" if f["kind"] == tb.GROUPED_WGRAD else "rows")
        x = a.data.float()
        if a_scale is not None:
            x = x * a_scale.repeat_interleave(128, 1)[:, : x.shape[1]]
        if rows is not None:
            x = x[rows.long().clamp_min(0)]
        at = offsets.tolist()
        for e, (lo, hi) in enumerate(zip(at, at[1:])):
            if f["kind"] == tb.GROUPED_WGRAD:
                c.data[e] = (x[lo:hi].t() @ b.data[lo:hi].float()).to(c.dtype)
                continue
            w = b.data[e].float()
            if b_scale is not None:
                s = b_scale[e].repeat_interleave(128, 0).repeat_interleave(128, 1)
                w = w * s[: w.shape[0], : w.shape[1]]
            y = x[lo:hi] @ (w if f["b_layout"] == tb.B_KN else w.t())
            if f["activation"] == tb.ACT_SWIGLU:
                y = torch.nn.functional.silu(y[:, : f["n"]]) * y[:, f["n"]:]
            c.data[lo:hi] = y.to(c.dtype)


def _stand_ins(log):
    def route(logits, ids, weights, slots, rows, offsets, renormalize=True, workspace=None):
        log.append("route")
        x = logits.data.float()
        top, at = x.topk(ids.shape[1], dim=1)
        ids.data.copy_(at)
        weights.data.copy_(torch.softmax(top, 1))
        pairs = sorted((int(at[t, j]), t, j) for t in range(at.shape[0])
                       for j in range(at.shape[1]))
        count = [0] * (x.shape[1] + 1)
        for s, (e, t, j) in enumerate(pairs):
            slots.data[t, j], rows.data[s] = s, t
            count[e + 1] += 1
        offsets.data.copy_(torch.tensor(count).cumsum(0))

    def route_backward(dweights, logits, ids, dlogits, renormalize=True):
        log.append("route_backward")
        w = torch.softmax(logits.data.gather(1, ids.long()), 1)
        d = w * (dweights.data - (w * dweights.data).sum(1, keepdim=True))
        dlogits.data.zero_().scatter_(1, ids.long(), d)

    def combine(y, slots, out, weights=None):
        log.append("combine")
        rows = y.data.float()[slots.long()]
        out.data.copy_((rows if weights is None else rows * weights.data[:, :, None]).sum(1))

    def combine_backward(dout, y, slots, weights, dy, dweights=None):
        log.append("combine_backward")
        d = dout.data.float()[:, None, :]
        dy.data[slots.long()] = (weights.data[:, :, None] * d).to(dy.dtype)
        if dweights is not None:
            log.append("dweights")
            dweights.data.copy_((y.data.float()[slots.long()] * d).sum(2))

    def quantize_f8(x, q, scale, block_rows=1):
        log.append("weights to 8 bits" if block_rows == 128 else "rows to 8 bits")
        *lead, n, k = x.shape
        v = torch.nn.functional.pad(x.data.float(), (0, -k % 128, 0, -n % block_rows))
        v = v.reshape(*lead, -(-n // block_rows), block_rows, -(-k // 128), 128)
        a = v.abs().amax((-3, -1)).clamp_min(2.0 ** -100)
        scale.data.copy_(a / 448)
        v = (v * (448 / a)[..., :, None, :, None]).flatten(-4, -3).flatten(-2, -1)
        q.data.copy_(v[..., :n, :k].to(torch.float8_e4m3fn))

    names = {n: getattr(tb, n) for n in dir(tb) if n.isupper()}
    desc = SimpleNamespace(from_config=lambda **f: _Desc(log, f))
    return SimpleNamespace(**names, GroupedDesc=desc, route=route, route_backward=route_backward,
                           combine=combine, combine_backward=combine_backward,
                           quantize_f8=quantize_f8, route_workspace_bytes=lambda *a: 64)


@pytest.fixture
def log(monkeypatch):
    out = []
    monkeypatch.setattr(moe_layer, "tb", _stand_ins(out))
    return out


def _layer(**sizes):
    base = dict(width=32, hidden=24, experts=4, top_k=2, device="cpu", seed=3)
    base.update(sizes)
    return moe_layer.ExpertLayer(**base)


def _x(layer, tokens=9, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((tokens, layer.width), generator=g).to(layer.dtype)


def _near(a, b):
    """8-bit operands are off by up to 2^-4 of a value, 3 roundings in all."""
    return float((a.float() - b.float()).norm() / b.float().norm()) < 3 * 2.0 ** -4


def test_8_bit_servers_follow_the_parameters(log):
    """Served in 8 bits, trained, served again: by a server of before and by a new
    one, after changes in place and after a parameter was replaced."""
    layer = _layer()
    x = _x(layer)
    before = layer.server(9, f8=True)
    assert _near(before.run(x), layer.server(9).run(x))
    with torch.no_grad():
        layer.up.mul_(-1.5)
    want = layer.server(9).run(x)
    assert _near(layer.server(9, f8=True).run(x), want)
    assert _near(before.run(x), want)
    layer.down = torch.flip(layer.down, (0,))
    want = layer.server(9).run(x)
    assert _near(layer.server(9, f8=True).run(x), want)
    assert _near(before.run(x), want)


def test_8_bit_weights_are_made_once_while_nothing_changes(log):
    layer = _layer()
    x = _x(layer)
    server = layer.server(9, f8=True)
    made = log.count("weights to 8 bits")
    held = [t.data_ptr() for t in server.weights]
    for _ in range(3):
        server.run(x)
    assert made == 2 and log.count("weights to 8 bits") == made
    # changed parameters go to the same buffers: a captured server reads those
    with torch.no_grad():
        layer.down.add_(1)
    server.run(x)
    assert log.count("weights to 8 bits") == 2 * made
    assert [t.data_ptr() for t in server.weights] == held


def test_8_bit_weights_of_changes_that_no_version_counts(log):
    """`.data` and inference tensors count no versions: a new server and `refresh`
    read what is there, and weights that count none are read every time."""
    layer = _layer()
    x = _x(layer)
    server = layer.server(9, f8=True)
    layer.up.data.mul_(-1.5)
    want = layer.server(9).run(x)
    assert _near(layer.server(9, f8=True).run(x), want)
    server.refresh()
    assert _near(server.run(x), want)
    with torch.inference_mode():
        layer = _layer()
        server = layer.server(9, f8=True)
        layer.up.mul_(-1.5)
        assert _near(server.run(x), layer.server(9).run(x))


def _train(layer, x, trained=("router", "up", "down")):
    for name in trained:
        setattr(layer, name, getattr(layer, name).detach().requires_grad_(True))
    return layer.train(x)


@pytest.mark.parametrize("trained", [("router",), ("up",), ("down",), ("router", "up", "down")])
@pytest.mark.parametrize("loss", [lambda out: out.float().sum(),
                                  lambda out: out.float().square().sum()])
def test_a_second_derivative_raises(log, trained, loss):
    """The gradients come from kernels that autograd sees nothing of: to differentiate
    them again is an error, not a term of zero, also beside terms that it does see and
    where the loss is linear, so that the output's gradient is a constant."""
    layer = _layer()
    out = _train(layer, _x(layer), trained)
    params = [getattr(layer, name) for name in trained]
    grads = torch.autograd.grad(loss(out), params, create_graph=True)
    penalty = sum(g.float().square().sum() for g in grads)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        torch.autograd.grad(penalty + loss(out), params, retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        penalty.backward()


def test_first_derivatives_with_a_graph_are_the_same(log):
    """Of the parameters whose gradients do not pass torch's silu, which has a
    formula of its own for gradients with a graph."""
    layer = _layer()
    out = _train(layer, _x(layer))
    params = [layer.router, layer.down]
    plain = torch.autograd.grad(out.float().sum(), params, retain_graph=True)
    graph = torch.autograd.grad(out.float().sum(), params, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))


@pytest.mark.parametrize("backward", [True, False])
def test_a_step_leaves_nothing_behind(log, monkeypatch, backward):
    """A step's routing and its buffers are freed with the step's graph, without
    Python's cycle collector."""
    alive = []

    class Routing(moe_layer.Routing):
        def __init__(self, *args):
            super().__init__(*args)
            alive.append(weakref.ref(self))
            alive.extend(weakref.ref(t) for t in vars(self).values()
                         if isinstance(t, torch.Tensor))

    monkeypatch.setattr(moe_layer, "Routing", Routing)
    layer = _layer()
    gc.collect()
    gc.disable()
    try:
        out = _train(layer, _x(layer))
        if backward:
            out.float().sum().backward()
        assert len(alive) > 4 and alive[0]() is not None
        del out
        assert [r for r in alive if r() is not None] == []
    finally:
        gc.enable()


@pytest.mark.parametrize("trained, want", [
    (("x",), ["route_backward", "combine_backward", "dweights", "rows", "rows", "combine"]),
    (("router",), ["route_backward", "combine_backward", "dweights"]),
    (("up",), ["combine_backward", "rows", "wgrad"]),
    (("down",), ["combine_backward", "wgrad"]),
    (("x", "router", "up", "down"), ["route_backward", "combine_backward", "dweights", "rows",
                                     "rows", "wgrad", "wgrad", "combine"])])
def test_only_the_gradients_asked_for_are_computed(log, trained, want):
    layer = _layer()
    leaves = {"x": _x(layer), "router": layer.router, "up": layer.up, "down": layer.down}
    for name in trained:
        leaves[name].requires_grad_(True)
    all_of = _layer()
    every = {"x": _x(layer), "router": all_of.router, "up": all_of.up, "down": all_of.down}
    for t in every.values():
        t.requires_grad_(True)
    all_of.train(every["x"]).float().sum().backward()
    out = layer.train(leaves["x"])
    log.clear()
    out.float().sum().backward()
    assert sorted(log) == sorted(want)
    for name in trained:
        assert torch.equal(leaves[name].grad, every[name].grad)


def test_8_bit_weights_that_the_caller_keeps(log):
    """Weights that the caller quantized are shared by servers, also of inference
    tensors, and made again when the caller says so."""
    with torch.inference_mode():
        layer = _layer()
        weights = layer.quantize()
        servers = [layer.server(n, f8=weights) for n in (9, 5)]
        for n, server in zip((9, 5), servers):
            server.run(_x(layer, n))
            assert all(a is b for a, b in zip(server.weights, weights))
        assert log.count("weights to 8 bits") == 2
        layer.up.mul_(-1.5)
        layer.quantize(weights)
        for n, server in zip((9, 5), servers):
            assert _near(server.run(_x(layer, n)), layer.server(n).run(_x(layer, n)))
        assert log.count("weights to 8 bits") == 4
