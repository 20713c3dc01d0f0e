"""A mixture-of-experts layer on the package's operators: an example.

    python -m mini_triton_nvgpu_v1_amd.moe_layer [--tokens T] [--steps N]

:class:`ExpertLayer` holds a router and gated experts, ``y = sum_j w_j
(silu(x G_e) * (x U_e)) D_e`` over a token's top_k experts e. ``serve`` computes
it with the activation fused into the first product, in 16 bits or with 8-bit
weights and activations, from the parameters as they are; ``train`` gives
torch's autograd the router, the products and the weighted sum with their
gradients. The program serves a decoding step and a prompt, trains a few steps,
and prints what each took.
"""
from __future__ import annotations

import argparse
import functools
import weakref

import torch

import mini_triton_nvgpu_v1_amd as tb

DTYPES = {torch.float16: tb.DTYPE_F16, torch.bfloat16: tb.DTYPE_BF16}


class Routing:
    """The buffers of one batch's routing; the weights are the caller's (in training
    they are an output that autograd's node holds on to, and that node the routing)."""

    def __init__(self, tokens: int, experts: int, top_k: int, device):
        i32 = torch.int32
        self.ids = torch.empty((tokens, top_k), dtype=i32, device=device)
        self.slots = torch.empty((tokens, top_k), dtype=i32, device=device)
        self.rows = torch.empty(tokens * top_k, dtype=i32, device=device)
        self.offsets = torch.empty(experts + 1, dtype=i32, device=device)
        size = tb.route_workspace_bytes(tokens, experts, top_k)
        self.workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None

    def run(self, logits, weights) -> None:
        tb.route(logits, self.ids, weights, self.slots, self.rows, self.offsets,
                 workspace=self.workspace)


class _Once(torch.autograd.Function):
    """The first `n` tensors, gradients made of the others: to go back through them raises."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the gradients of an expert layer cannot be differentiated again")


def _once(backward):
    """A backward pass of kernels that autograd sees nothing of. Where its gradients get
    a graph of their own (create_graph), that graph ends in an error at all they were
    made of; torch's once_differentiable lets them pass as constants where the
    incoming gradient is one, and where no leaf that is asked for lies behind it."""

    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        at = [i for i, g in enumerate(out) if g is not None]
        tied = _Once.apply(len(at), *(out[i] for i in at), *ctx.saved_tensors, *grads)
        return tuple(tied[at.index(i)] if i in at else None for i in range(len(out)))

    return run


class _Route(torch.autograd.Function):
    """logits -> weights, and the routing's order in `routing`."""

    @staticmethod
    def forward(ctx, logits, routing):
        weights = torch.empty(routing.ids.shape, device=logits.device)
        routing.run(logits, weights)
        ctx.save_for_backward(logits)
        ctx.ids = routing.ids
        return weights

    @staticmethod
    @_once
    def backward(ctx, dweights):
        (logits,) = ctx.saved_tensors
        dlogits = torch.empty_like(logits)
        tb.route_backward(dweights.contiguous(), logits, ctx.ids, dlogits)
        return dlogits, None


class _Product(torch.autograd.Function):
    """x (rows gathered by `rows`, or slot by slot) times each slot's expert's
    weights (experts x k x n)."""

    @staticmethod
    def forward(ctx, x, w, routing, gather):
        groups, k, n = w.shape
        code = DTYPES[x.dtype]
        slots = routing.rows.numel()
        rows = routing.rows if gather else None
        # slots past the last pair (too few experts left for a token) stay zero
        y = torch.zeros((slots, n), dtype=x.dtype, device=x.device)
        tb.GroupedDesc.from_config(groups=groups, n=n, k=k, dtype=code, c_dtype=code).launch(
            x, w, y, offsets=routing.offsets, rows=rows)
        ctx.save_for_backward(x, w)
        ctx.routing, ctx.gather = routing, gather
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        groups, k, n = w.shape
        code, r = DTYPES[x.dtype], ctx.routing
        dy = dy.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            # of the rows: the product with the transposed weights, slot by slot
            dx = torch.zeros((dy.shape[0], k), dtype=x.dtype, device=x.device)
            tb.GroupedDesc.from_config(groups=groups, n=k, k=n, dtype=code, c_dtype=code,
                                       b_layout=tb.B_NK).launch(dy, w, dx, offsets=r.offsets)
            if ctx.gather:
                drows, dx = dx, torch.empty_like(x)  # a token's rows, each with weight one
                tb.combine(drows, r.slots, dx)
        if ctx.needs_input_grad[1]:
            dw = torch.empty_like(w)
            tb.GroupedDesc.from_config(kind=tb.GROUPED_WGRAD, groups=groups, n=n, k=k,
                                       dtype=code, c_dtype=code).launch(
                x, dy, dw, offsets=r.offsets, rows=r.rows if ctx.gather else None)
        return dx, dw, None, None


class _Combine(torch.autograd.Function):
    """The weighted sum of each token's rows."""

    @staticmethod
    def forward(ctx, y, weights, routing):
        out = torch.empty((weights.shape[0], y.shape[1]), dtype=y.dtype, device=y.device)
        tb.combine(y, routing.slots, out, weights=weights)
        ctx.save_for_backward(y, weights)
        ctx.routing = routing
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        y, weights = ctx.saved_tensors
        dy = torch.zeros_like(y)
        dw = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        tb.combine_backward(dout.contiguous(), y, ctx.routing.slots, weights, dy, dw)
        return dy if ctx.needs_input_grad[0] else None, dw, None


class ExpertLayer:
    """Router (width x experts, f32) and experts: `up` experts x width x 2 hidden,
    the gate's columns first, and `down` experts x hidden x width."""

    def __init__(self, width: int, hidden: int, experts: int, top_k: int,
                 dtype=torch.bfloat16, device="cuda", seed: int = 0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def made(*shape, dt=dtype):
            w = torch.randn(shape, generator=g, device=device) * shape[-2] ** -0.5
            return w.to(dt)

        self.width, self.hidden, self.experts, self.top_k = width, hidden, experts, top_k
        self.dtype = dtype
        self.router = made(width, experts, dt=torch.float32)
        self.up = made(experts, width, 2 * hidden)
        self.down = made(experts, hidden, width)

    def parameters(self):
        return [self.router, self.up, self.down]

    def train(self, x):
        """The layer for autograd; the activation is torch's."""
        routing = Routing(x.shape[0], self.experts, self.top_k, x.device)
        weights = _Route.apply(x.float() @ self.router, routing)
        h = _Product.apply(x, self.up, routing, True)
        gate, u = h.chunk(2, dim=1)
        y = _Product.apply(torch.nn.functional.silu(gate) * u, self.down, routing, False)
        return _Combine.apply(y, weights, routing)

    def quantize(self, out: list | None = None) -> list:
        """The experts' weights as they are, in 8 bits, rows of the output contiguous:
        up, its scales, down, its scales. `out`: what an earlier call gave, written
        again."""
        made = []
        for i, w in enumerate((self.up, self.down)):
            w = w.transpose(1, 2).contiguous()
            e, n, k = w.shape
            q, s = out[2 * i:2 * i + 2] if out else (
                torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device),
                torch.empty((e, -(-n // 128), -(-k // 128)), device=w.device))
            tb.quantize_f8(w, q, s, block_rows=128)
            made += [q, s]
        return made

    def server(self, tokens: int, f8: bool | list = False) -> "Server":
        return Server(self, tokens, f8)


def _state(w):
    """What tells a parameter's values apart: the tensor and its count of changes
    (None: inference tensors have none)."""
    return weakref.ref(w), None if w.is_inference() else w._version


class Server:
    """Descriptors and buffers for batches of `tokens` tokens; `run` is the layer.

    `f8`: the server holds the weights in 8 bits, and `run` makes them again, in
    place, when a parameter was replaced or changed. Of changes through `.data` or
    other libraries' pointers torch counts no version: `refresh` says that there
    were some. Inference tensors have no version at all: from those every `run`
    makes the weights again. Weights that the caller quantized, `f8` what
    ExpertLayer.quantize gave, can be shared by servers and stay as they are until
    it is given them again."""

    def __init__(self, layer: ExpertLayer, tokens: int, f8: bool | list):
        dev, code = layer.up.device, DTYPES[layer.dtype]
        self.layer, self.f8 = layer, bool(f8)
        self.weights, self._of = (f8, None) if isinstance(f8, list) else (None, ())
        slots = tokens * layer.top_k
        self.routing = Routing(tokens, layer.experts, layer.top_k, dev)
        self.route_weights = torch.empty((tokens, layer.top_k), device=dev)
        self.h = torch.empty((slots, layer.hidden), dtype=layer.dtype, device=dev)
        # slots without a pair are read by no token
        self.y = torch.empty((slots, layer.width), dtype=layer.dtype, device=dev)
        self.out = torch.empty((tokens, layer.width), dtype=layer.dtype, device=dev)
        kind = dict(groups=layer.experts, c_dtype=code, dtype=tb.DTYPE_F8E4M3 if f8 else code,
                    b_layout=tb.B_NK if f8 else tb.B_KN)
        self.first = tb.GroupedDesc.from_config(n=layer.hidden, k=layer.width,
                                                activation=tb.ACT_SWIGLU, **kind)
        self.second = tb.GroupedDesc.from_config(n=layer.width, k=layer.hidden, **kind)
        if f8:
            def e4m3(rows, cols):
                return (torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=dev),
                        torch.empty((rows, -(-cols // 128)), device=dev))

            self.xq, self.hq = e4m3(tokens, layer.width), e4m3(slots, layer.hidden)
            if self.weights is None:
                self.refresh()

    def refresh(self) -> None:
        """The parameters as they are now, in 8 bits (16-bit servers read them anyway)."""
        if not self.f8:
            return
        self.weights = self.layer.quantize(self.weights)
        if self._of is not None:
            self._of = [_state(w) for w in (self.layer.up, self.layer.down)]

    def _changed(self) -> bool:
        return self._of is not None and any(
            ref() is not w or version is None or version != w._version
            for w, (ref, version) in zip((self.layer.up, self.layer.down), self._of))

    def run(self, x):
        layer, r = self.layer, self.routing
        r.run(x.float() @ layer.router, self.route_weights)
        if self.f8:
            if self._changed():
                self.refresh()
            up, up_scale, down, down_scale = self.weights
            tb.quantize_f8(x, *self.xq)
            self.first.launch(self.xq[0], up, self.h, offsets=r.offsets, rows=r.rows,
                              a_scale=self.xq[1], b_scale=up_scale)
            tb.quantize_f8(self.h, *self.hq)
            self.second.launch(self.hq[0], down, self.y, offsets=r.offsets,
                               a_scale=self.hq[1], b_scale=down_scale)
        else:
            self.first.launch(x, layer.up, self.h, offsets=r.offsets, rows=r.rows)
            self.second.launch(self.h, layer.down, self.y, offsets=r.offsets)
        tb.combine(self.y, r.slots, self.out, weights=self.route_weights)
        return self.out


def _us(f, n: int = 20) -> float:
    for _ in range(3):
        f()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for _ in range(n):
        f()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / n * 1e3


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=5)
    args = ap.parse_args()
    layer = ExpertLayer(width=2048, hidden=1024, experts=64, top_k=6)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    weights8 = layer.quantize()
    for tokens in (13, args.tokens):
        x = torch.randn((tokens, layer.width), generator=g, device="cuda").to(layer.dtype)
        plain, f8 = layer.server(tokens), layer.server(tokens, f8=weights8)
        a, b = plain.run(x).float(), f8.run(x).float()
        off = float((a - b).norm() / a.norm())
        print(f"serving {tokens} tokens: {_us(lambda: plain.run(x)):.0f} us in 16 bits, "
              f"{_us(lambda: f8.run(x)):.0f} us in 8 bits, which differ by {off:.3f}")
    x = torch.randn((args.tokens, layer.width), generator=g, device="cuda").to(layer.dtype)
    target = torch.randn(x.shape, generator=g, device="cuda")
    for p in layer.parameters():
        p.requires_grad_(True)
    for step in range(args.steps):
        for p in layer.parameters():
            p.grad = None
        loss = (layer.train(x).float() - target).square().mean()
        loss.backward()
        with torch.no_grad():
            # each parameter moves by 1 % of its size against its gradient
            for p in layer.parameters():
                d = p.grad.float()
                size = p.float().square().mean().sqrt()
                p -= (0.01 * size * d / d.square().mean().sqrt()).to(p.dtype)
        print(f"step {step}: loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
