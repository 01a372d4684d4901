"""A transformer's feed-forward sublayer with experts on the operators of ``tiramisu_amd.operators``: a router sends every token to k of many small gated layers, whose
results, weighted, are added to the residual stream.  Trained in 16 bits, served in 16 or in 8.

    sum = x + residual,  n = rms_norm(sum),  the k experts e of the largest n router^T, w their softmax,  y = sum + the sum over them of w_e (silu(n gate_e^T) * (n up_e^T)) down_e^T

``python -m tiramisu_amd.expert_feed_forward`` trains one on random data for some steps, then serves tokens with what it learnt and says how far 8 bits are from 16.  (The same
forward pass as a Tiramisu program: tiramisu_amd/programs/expert_feed_forward.cpp.)
"""
from typing import NamedTuple

import torch

from . import operators


class Kept(NamedTuple):
    """What a training step's forward pass keeps for its backward pass."""
    sum: torch.Tensor
    rstd: torch.Tensor
    n: torch.Tensor
    logits: torch.Tensor
    route: operators.Route
    gate: torch.Tensor
    up: torch.Tensor
    h: torch.Tensor
    rows: torch.Tensor                      # of the experts, ahead of their weights


class ExpertFeedForward:
    """Weights of one sublayer, on the GPU: ``norm`` [hidden], ``router`` [experts, hidden], ``gate`` and ``up`` [experts, inner, hidden], ``down`` [experts, hidden, inner]."""

    NAMES = ("norm", "router", "gate", "up", "down")

    def __init__(self, hidden, inner, experts, k, dtype=torch.bfloat16, device="cuda", generator=None, activation="silu", eps=1e-6):
        self.k, self.activation, self.eps = k, activation, eps
        self.norm = torch.ones(hidden, dtype=dtype, device=device)
        self.router, self.gate, self.up, self.down = [(torch.randn(shape, device=device, generator=generator) * shape[-1] ** -0.5).to(dtype)
                                                      for shape in ((experts, hidden), (experts, inner, hidden), (experts, inner, hidden), (experts, hidden, inner))]

    def forward(self, x, residual):
        """(y, what ``backward`` needs)"""
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps, keep_rstd=True)
        logits = operators.linear(n.y, self.router).y
        r = operators.route(logits, self.k)
        g = operators.grouped_gated_linear(n.y, self.gate, self.up, r.offsets, rows=r.rows, activation=self.activation, keep_pre=True)
        rows = operators.grouped_linear(g.h, self.down, r.offsets)
        y = operators.combine(rows, r.places, weights=r.weights, residual=n.sum)
        return y, Kept(n.sum, n.rstd, n.y, logits, r, g.gate, g.up, g.h, rows)

    def backward(self, dy, kept):
        """(gradient of x and of the residual alike, gradients of the weights by name)"""
        r = kept.route
        c = operators.combine_backward(dy, kept.rows, r.places, r.weights, r.rows)
        down = operators.grouped_linear_backward(c.dx, kept.h, self.down, r.offsets)
        gated = operators.grouped_gated_linear_backward(down.dx, kept.n, self.gate, self.up, kept.gate, kept.up, r.offsets, rows=r.rows, activation=self.activation)
        router = operators.linear_backward(operators.route_backward(c.dweights, kept.logits, r.experts), kept.n, self.router)
        dn = operators.combine(gated.dx, r.places, residual=router.dx)
        norm = operators.rms_norm_backward(dn, kept.sum, self.norm, kept.rstd, dsum=dy)
        return norm.dx, {"norm": norm.dweight, "router": router.dweight, "gate": gated.dgate_weight, "up": gated.dup_weight, "down": down.dweight}

    def serve(self, x, residual):
        """y alone; nothing is kept."""
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps)
        r = operators.route(operators.linear(n.y, self.router).y, self.k)
        h = operators.grouped_gated_linear(n.y, self.gate, self.up, r.offsets, rows=r.rows, activation=self.activation).h
        return operators.combine(operators.grouped_linear(h, self.down, r.offsets), r.places, weights=r.weights, residual=n.sum)

    def in_8_bits(self):
        """The sublayer with its experts' matrices as 8-bit rows with scales, laid out once."""
        return EightBitExperts(self)


class EightBitExperts:
    """Serves an ``ExpertFeedForward`` with 8-bit experts; the router stays in 16 bits, so that it chooses as it did in training."""

    def __init__(self, layer):
        self.norm, self.router, self.k, self.activation, self.eps, self.dtype = layer.norm, layer.router, layer.k, layer.activation, layer.eps, layer.norm.dtype
        self.gate, self.up, self.down = [operators.quantize_rows(w) for w in (layer.gate, layer.up, layer.down)]

    def serve(self, x, residual):
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps)
        r = operators.route(operators.linear(n.y, self.router).y, self.k)
        q = operators.quantize_rows(n.y)
        h = operators.grouped_gated_linear(q.q, self.gate.q, self.up.q, r.offsets, rows=r.rows, activation=self.activation, x_scale=q.scale, gate_scale=self.gate.scale,
                                           up_scale=self.up.scale, dtype=self.dtype).h
        q = operators.quantize_rows(h)
        rows = operators.grouped_linear(q.q, self.down.q, r.offsets, x_scale=q.scale, weight_scale=self.down.scale, dtype=self.dtype)
        return operators.combine(rows, r.places, weights=r.weights, residual=n.sum)


def disturbed(layer, by, generator=None):
    """The layer with random numbers of `by` times its weights' size added to them; the router as it is."""
    experts, inner, hidden = layer.gate.shape
    other = ExpertFeedForward(hidden, inner, experts, layer.k, layer.norm.dtype, layer.norm.device, generator, layer.activation, layer.eps)
    other.router.copy_(layer.router)
    for name in ("gate", "up", "down"):
        getattr(other, name).mul_(by).add_(getattr(layer, name))
    return other


def train(layer, teacher, steps, tokens, rate=0.1, generator=None):
    """Fits the layer to another one on random tokens, by plain gradient descent on 32-bit copies of the weights; the mean squared errors, step by
    step.  (An expert sees k tokens of every `experts`: its rate is as much larger.)"""
    experts, _, hidden = layer.gate.shape
    wide = {name: getattr(layer, name).float() for name in layer.NAMES}
    errors = []
    for _ in range(steps):
        x, residual = [torch.randn((tokens, hidden), device=layer.norm.device, generator=generator).to(layer.norm.dtype) for _ in range(2)]
        y, kept = layer.forward(x, residual)
        off = y.float() - teacher.serve(x, residual).float()
        errors.append(off.square().mean())
        _, gradients = layer.backward((off * (2.0 / tokens)).to(y.dtype), kept)
        for name in layer.NAMES:
            wide[name] -= rate * (1.0 if name in ("norm", "router") else experts / layer.k) * gradients[name].float()
            getattr(layer, name).copy_(wide[name])
    return [float(e) for e in errors]


def main():
    generator = torch.Generator(device="cuda")
    generator.manual_seed(0)
    teacher = ExpertFeedForward(1024, 512, 32, 4, generator=generator)
    layer = disturbed(teacher, 0.5, generator)
    errors = train(layer, teacher, 60, 4096, generator=generator)
    print("mean squared error: %.4f at first, %.4f after %d steps" % (errors[0], errors[-1], len(errors)))
    small = layer.in_8_bits()
    for tokens in (1, 16, 2048):
        x, residual = [torch.randn((tokens, 1024), device="cuda", generator=generator).to(torch.bfloat16) for _ in range(2)]
        y, y8 = layer.serve(x, residual).float(), small.serve(x, residual).float()
        branch = y - (x + residual).float()
        print("%4d tokens: 8 bits are %.3f of the sublayer's own part away from 16" % (tokens, float((y8 - y).norm() / branch.norm())))


if __name__ == "__main__":
    main()
