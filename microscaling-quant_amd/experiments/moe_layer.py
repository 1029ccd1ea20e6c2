"""A mixture-of-experts layer on packed MX weights, from the router's logits to the summed output; not in the reference.

    layer = MoELayer.from_weights(router, gate_up, down, shared_up, shared_down, top_k=2)     float weights, packed here
    y = layer(x)                                   tokens x D
    grad = layer.router_gradient(x, grad_y)        of the router's weight: routing and combining are differentiable

    python -m experiments.moe_layer --tokens 256 --width 1024 --hidden 2816 --experts 8 --fmt MXFP8_E4M3

prints how far the layer is from the same layer on the dequantized weights in float32, and what a call takes.
"""
import argparse
import time

import torch

from mxq import nn, packed

__all__ = ["MoELayer", "main"]


class MoELayer:
    """router: E x D.  gate_up: E x 2 F x D, gates first; down: E x D x F; shared_up (2 S x D) and shared_down (D x S):
    an expert that every token takes, or None.  All but the router are (codes, scales) of `fmt`."""

    def __init__(self, router, gate_up, down, shared_up=None, shared_down=None, *, fmt="MXFP8_E4M3", top_k=2, **routing):
        self.router, self.gate_up, self.down = router, gate_up, down
        self.shared_up, self.shared_down = shared_up, shared_down
        self.fmt, self.top_k, self.routing = fmt, top_k, routing

    @classmethod
    def from_weights(cls, router, gate_up, down, shared_up=None, shared_down=None, *, fmt="MXFP8_E4M3", **more):
        pack = lambda w: None if w is None else packed.quantize(w, fmt, axis=-1)
        return cls(router, pack(gate_up), pack(down), pack(shared_up), pack(shared_down), fmt=fmt, **more)

    def _experts(self, x, experts):
        plan = nn.dispatch(experts, self.router.shape[0])
        h = nn.expert_linear(x, *self.gate_up, self.fmt, plan, activation="silu", gated=True)
        y = nn.expert_linear(h, *self.down, self.fmt, plan, sorted_rows=True)
        shared = None
        if self.shared_up is not None:
            s = nn.packed_linear(x, *self.shared_up, self.fmt, activation="silu", gated=True)
            shared = nn.packed_linear(s, *self.shared_down, self.fmt)
        return plan, y, shared

    def __call__(self, x):
        weights, experts = nn.route((x @ self.router.t()).float(), self.top_k, **self.routing)
        plan, y, shared = self._experts(x, experts)
        return nn.combine(y, weights, plan, residual=shared)

    def router_gradient(self, x, grad_y):
        """The gradient of the router's weight; the experts' weights are bytes and have none, nor do their
        products have one of x, so that a call refuses an x that asks for it."""
        router, x = self.router.detach().requires_grad_(), x.detach()
        weights, experts = nn.route((x @ router.t()).float(), self.top_k, **self.routing)
        plan, y, shared = self._experts(x, experts)
        return torch.autograd.grad(nn.combine(y, weights, plan, residual=shared), router, grad_y)[0]


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 256), ("width", 1024), ("hidden", 2816), ("experts", 8), ("top-k", 2), ("shared", 1024)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--fmt", default="MXFP8_E4M3")
    a = p.parse_args(argv)
    dev, gen = "cuda", torch.Generator("cuda").manual_seed(0)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=dev) * shape[-1] ** -0.5
    floats = (normal(a.experts, 2 * a.hidden, a.width), normal(a.experts, a.width, a.hidden),
              normal(2 * a.shared, a.width), normal(a.width, a.shared))
    layer = MoELayer.from_weights(normal(a.experts, a.width).bfloat16(), *floats, fmt=a.fmt, top_k=a.top_k)
    x = (normal(a.tokens, a.width) * a.width ** 0.5).bfloat16()
    y = layer(x)

    # the same choices on the dequantized weights, float32, an expert at a time
    bytes_of = (layer.gate_up, layer.down, layer.shared_up, layer.shared_down)
    up, down, s_up, s_down = (packed.dequantize(*w, a.fmt, axis=-1) for w in bytes_of)
    weights, experts = nn.route((x @ layer.router.t()).float(), a.top_k)
    gated = lambda z: torch.nn.functional.silu(z[:, :z.shape[1] // 2]) * z[:, z.shape[1] // 2:]
    want = gated(x.float() @ s_up.t()) @ s_down.t()
    for t, j in torch.nonzero(experts >= 0).tolist():
        e = int(experts[t, j])
        want[t] += weights[t, j] * (gated(x[t:t + 1].float() @ up[e].t()) @ down[e].t())[0]
    off = float((y.float() - want).norm() / want.norm())

    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(20):
        layer(x)
    torch.cuda.synchronize()
    us = (time.perf_counter() - start) / 20 * 1e6
    print(f"{a.tokens} tokens, {a.experts} experts of {a.width} x {a.hidden} in {a.fmt}: {us:.1f} us a call, "
          f"{off:.2e} from float32 on the dequantized weights")
    return {"us": us, "relative": off}


if __name__ == "__main__":
    main()
