"""A transformer's feed-forward sublayer on the operators of ``tiramisu_amd.operators``: trained in 16 bits, served in 16 or in 8.

    sum = x + residual,  n = rms_norm(sum),  h = silu(n gate^T) * (n up^T),  y = sum + h down^T

``python -m tiramisu_amd.feed_forward`` trains one on random data for some steps, then serves tokens with what it learnt and says how far 8 bits
are from 16.  (The same forward pass as a Tiramisu program: tiramisu_amd/programs/feed_forward.cpp.)
"""
from typing import NamedTuple

import torch

from . import operators


class Kept(NamedTuple):
    """What a training step's forward pass keeps for its backward pass."""
    sum: torch.Tensor
    rstd: torch.Tensor
    n: torch.Tensor
    gate: torch.Tensor
    up: torch.Tensor
    h: torch.Tensor


class FeedForward:
    """Weights of one sublayer, on the GPU: ``norm`` [hidden], ``gate`` and ``up`` [inner, hidden], ``down`` [hidden, inner]."""

    NAMES = ("norm", "gate", "up", "down")

    def __init__(self, hidden, inner, dtype=torch.bfloat16, device="cuda", generator=None, activation="silu", eps=1e-6):
        self.activation, self.eps = activation, eps
        self.norm = torch.ones(hidden, dtype=dtype, device=device)
        self.gate, self.up, self.down = [(torch.randn(shape, device=device, generator=generator) * shape[1] ** -0.5).to(dtype)
                                         for shape in ((inner, hidden), (inner, hidden), (hidden, inner))]

    def forward(self, x, residual):
        """(y, what ``backward`` needs)"""
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps, keep_rstd=True)
        g = operators.gated_linear(n.y, self.gate, self.up, activation=self.activation, keep_pre=True)
        y = operators.linear(g.h, self.down, residual=n.sum).y
        return y, Kept(n.sum, n.rstd, n.y, g.gate, g.up, g.h)

    def backward(self, dy, kept):
        """(gradient of x and of the residual alike, gradients of the weights by name)"""
        down = operators.linear_backward(dy, kept.h, self.down)
        gated = operators.gated_linear_backward(down.dx, kept.n, self.gate, self.up, kept.gate, kept.up, activation=self.activation)
        norm = operators.rms_norm_backward(gated.dx, kept.sum, self.norm, kept.rstd, dsum=dy)
        return norm.dx, {"norm": norm.dweight, "gate": gated.dgate_weight, "up": gated.dup_weight, "down": down.dweight}

    def serve(self, x, residual):
        """y alone, and the sum that the next sublayer's residual stream begins with; nothing is kept."""
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps)
        h = operators.gated_linear(n.y, self.gate, self.up, activation=self.activation).h
        return operators.linear(h, self.down, residual=n.sum).y

    def in_8_bits(self):
        """The sublayer with its matrices as 8-bit rows with scales, laid out once."""
        return EightBitFeedForward(self)


class EightBitFeedForward:
    """Serves a ``FeedForward`` with 8-bit matrices: the norm's results leave it in 8 bits, the gated layer's are brought to 8 bits ahead of the down
    projection."""

    def __init__(self, layer):
        self.norm, self.activation, self.eps, self.dtype = layer.norm, layer.activation, layer.eps, layer.norm.dtype
        self.gate, self.up, self.down = [operators.quantize_rows(w) for w in (layer.gate, layer.up, layer.down)]

    def serve(self, x, residual):
        n = operators.rms_norm(x, self.norm, residual=residual, eps=self.eps, eight_bit=True)
        h = operators.gated_linear(n.y, self.gate.q, self.up.q, activation=self.activation, x_scale=n.scale, gate_scale=self.gate.scale,
                                   up_scale=self.up.scale, dtype=self.dtype).h
        h = operators.quantize_rows(h)
        return operators.linear(h.q, self.down.q, residual=n.sum, x_scale=h.scale, weight_scale=self.down.scale, dtype=self.dtype).y


def disturbed(layer, by, generator=None):
    """The layer with random numbers of `by` times its weights' size added to them."""
    other = FeedForward(layer.gate.shape[1], layer.gate.shape[0], layer.norm.dtype, layer.norm.device, generator, layer.activation, layer.eps)
    for name in ("gate", "up", "down"):
        getattr(other, name).mul_(by).add_(getattr(layer, name))
    return other


def train(layer, teacher, steps, tokens, rate=0.1, generator=None):
    """Fits the layer to another one on random tokens, by plain gradient descent on 32-bit copies of the weights; the mean squared errors, step by
    step."""
    hidden = layer.gate.shape[1]
    wide = {name: getattr(layer, name).float() for name in layer.NAMES}
    errors = []
    for _ in range(steps):
        x, residual = [torch.randn((tokens, hidden), device=layer.norm.device, generator=generator).to(layer.norm.dtype) for _ in range(2)]
        y, kept = layer.forward(x, residual)
        off = y.float() - teacher.serve(x, residual).float()
        errors.append(off.square().mean())
        _, gradients = layer.backward((off * (2.0 / tokens)).to(y.dtype), kept)
        for name in layer.NAMES:
            wide[name] -= rate * gradients[name].float()
            getattr(layer, name).copy_(wide[name])
    return [float(e) for e in errors]


def main():
    generator = torch.Generator(device="cuda")
    generator.manual_seed(0)
    teacher = FeedForward(1024, 4096, generator=generator)
    layer = disturbed(teacher, 0.5, generator)
    errors = train(layer, teacher, 60, 2048, generator=generator)
    print("mean squared error: %.4f at first, %.4f after %d steps" % (errors[0], errors[-1], len(errors)))
    small = layer.in_8_bits()
    for tokens in (1, 16, 2048):
        x, residual = [torch.randn((tokens, 1024), device="cuda", generator=generator).to(torch.bfloat16) for _ in range(2)]
        y, y8 = layer.serve(x, residual).float(), small.serve(x, residual).float()
        branch = y - (x + residual).float()
        print("%4d tokens: 8 bits are %.3f of the sublayer's own part away from 16" % (tokens, float((y8 - y).norm() / branch.norm())))


if __name__ == "__main__":
    main()
