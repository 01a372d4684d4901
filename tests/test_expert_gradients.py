"""Gradients of a whole feed-forward sublayer with experts against 64-bit autograd of the same sublayer with the router's choice held, element by element and by their norm.

Tolerances follow every stored intermediate through the sublayer: a number is carried with the standard deviation of what the operators' are off it.  Storing is off by at most u of itself (u of the
type: half a step), evenly spread, so by u / sqrt 3 in the root mean square; different numbers' roundings do not know of each other, so that squares add up in products and sums.  32-bit sums add
2 (n + 8) 2^-24 of the magnitudes for n terms (test_operators.py); silu has slopes of at most 1.1 and its slope slopes of at most 1/2; a softmax weight moves by itself times what its logit and
the weights' mean of all move.  An error that arrives along several ways, four at most (through gate and up, the weight and the row), adds up to twice of what its squares say.  An element may be off by ten standard deviations: five, which one number in
two million exceeds, and twice.  The norm of all elements' errors may be three of theirs from 30 tokens on: twice, and half as much again as its square varies by a quarter where only the tokens' errors (of a router's choice, which
a whole row of gradients shares) do not know of each other.
That these are no looser than a mistake is checked on the CPU: with the router's term, an expert or the branch left out, or a factor, the exact gradients themselves leave them."""
import math

import pytest
import torch

from test_operators import LEAST, ROUNDOFF
from tiramisu_amd import expert_feed_forward

EPS = 1e-6


class Number:
    """64-bit numbers and the standard deviation of the operators' from them"""

    def __init__(self, value, off=None):
        self.value, self.off = value, torch.zeros_like(value) if off is None else off

    def __getitem__(self, at):
        return Number(self.value[at], self.off[at])

    def t(self):
        return Number(self.value.t(), self.off.t())

    def __add__(self, other):
        return Number(self.value + other.value, torch.hypot(self.off, other.off) + 2.0 ** -23 * (self.value.abs() + other.value.abs()))

    def __neg__(self):
        return Number(-self.value, self.off)

    def __mul__(self, other):
        return Number(self.value * other.value, torch.hypot(self.off * other.value.abs(), self.value.abs() * other.off) + self.off * other.off + 2.0 ** -23 * (self.value * other.value).abs())

    def __matmul__(self, other):
        n, squares = self.value.shape[-1], self.off.square() @ (other.value.square() + other.off.square()) + self.value.square() @ other.off.square()
        return Number(self.value @ other.value, squares.sqrt() + 2 * (n + 8) * 2.0 ** -24 * (self.value.abs() @ other.value.abs()))

    def sum(self, dim):
        n = self.value.shape[dim]
        return Number(self.value.sum(dim, keepdim=True), self.off.square().sum(dim, keepdim=True).sqrt() + 2 * (n + 8) * 2.0 ** -24 * self.value.abs().sum(dim, keepdim=True))

    def stored(self, dtype):
        return Number(self.value, torch.hypot(self.off, ROUNDOFF[dtype] / math.sqrt(3) * self.value.abs()) + LEAST[dtype])


def silu(z):
    return Number(z.value * torch.sigmoid(z.value), 1.1 * z.off + 2.0 ** -22 * (z.value.abs() + 1))


def silu_slope(z):
    s = torch.sigmoid(z.value)
    return Number(s * (1 + z.value * (1 - s)), 0.5 * z.off + 16 * 2.0 ** -24 * (z.value.abs() + 1))


def followed(weights, x, residual, experts, dy, dtype, of_sublayer):
    """Gradients of x and of the weights by name, as Numbers.  of_sublayer: with the norm ahead and the residual stream's gradient added, as ExpertFeedForward has them; else of the branch."""
    w = {name: Number(t) for name, t in weights.items()}
    dy = Number(dy)
    if of_sublayer:
        total = Number(x + residual)
        rstd = torch.rsqrt(total.value.square().mean(1, keepdim=True) + EPS)
        rstd = Number(rstd, (x.shape[1] + 16) * 2.0 ** -24 * rstd)
        n = (total * rstd * w["norm"]).stored(dtype)
        total = total.stored(dtype)
    else:
        n = Number(x)
    logits = (n @ w["router"].t()).stored(dtype)
    chosen = Number(logits.value.gather(1, experts), logits.off.gather(1, experts))
    share = torch.softmax(chosen.value, 1)
    share = Number(share, share * (torch.hypot(chosen.off, (share * chosen.off).square().sum(1, keepdim=True).sqrt()) + 2.0 ** -20))
    T, k = experts.shape
    dshare, dn = Number(torch.zeros_like(share.value)), Number(torch.zeros_like(n.value))
    gradients = {name: Number(torch.zeros_like(t)) for name, t in weights.items()}

    def put(where, at, numbers):
        where.value[at], where.off[at] = numbers.value, numbers.off

    of_places = Number(torch.zeros((T, k, n.value.shape[1]), dtype=torch.float64, device=x.device))
    for e in range(len(weights["gate"])):
        token, rank = torch.nonzero(experts == e, as_tuple=True)
        if len(token) == 0:
            continue
        rows = n[token]
        gate, up = rows @ w["gate"][e].t(), rows @ w["up"][e].t()
        h = (silu(gate) * up).stored(dtype)
        gate, up = gate.stored(dtype), up.stored(dtype)
        out = (h @ w["down"][e].t()).stored(dtype)
        put(dshare, (token, rank), (dy[token] * out).sum(1)[:, 0])
        dout = (share[token, rank][:, None] * dy[token]).stored(dtype)
        put(gradients["down"], e, (dout.t() @ h).stored(dtype))
        dh = (dout @ w["down"][e]).stored(dtype)
        dgate, dup = (dh * up * silu_slope(gate)).stored(dtype), (dh * silu(gate)).stored(dtype)
        put(gradients["gate"], e, (dgate.t() @ rows).stored(dtype))
        put(gradients["up"], e, (dup.t() @ rows).stored(dtype))
        put(of_places, (token, rank), (dgate @ w["gate"][e] + dup @ w["up"][e]).stored(dtype))
    dchosen = share * (dshare + -((share * dshare).sum(1)))
    dlogits = Number(torch.zeros_like(logits.value).scatter(1, experts, dchosen.value), torch.zeros_like(logits.value).scatter(1, experts, dchosen.off)).stored(dtype)
    gradients["router"] = (dlogits.t() @ n).stored(dtype)
    dn = ((dlogits @ w["router"]).stored(dtype) + of_places.sum(1)[:, 0]).stored(dtype)
    if not of_sublayer:
        return dict(gradients, x=dn)
    hat, scaled = total * rstd, dn * w["norm"]
    gradients["norm"] = ((dn * hat).sum(0)[0]).stored(dtype)
    mean = (scaled * hat).sum(1)
    mean = Number(mean.value / x.shape[1], mean.off / x.shape[1])
    dx = (rstd * (scaled + -(hat * mean)) + dy).stored(dtype)
    return dict(gradients, x=dx)


def exact(weights, x, residual, experts, dy, of_sublayer, router_counts=True):
    """The same by autograd"""
    at = {name: t.clone().requires_grad_() for name, t in dict(weights, x=x).items()}
    n = total = at["x"]
    if of_sublayer:
        total = at["x"] + residual
        n = total * torch.rsqrt(total.square().mean(1, keepdim=True) + EPS) * at["norm"]
    share = torch.softmax((n @ at["router"].t()).gather(1, experts), 1)
    if not router_counts:
        share = share.detach()
    y = total if of_sublayer else 0
    for e in range(len(weights["gate"])):
        out = (torch.nn.functional.silu(n @ at["gate"][e].t()) * (n @ at["up"][e].t())) @ at["down"][e].t()
        y = y + (share * (experts == e)).sum(1, keepdim=True) * out
    names = [name for name in at if (name != "norm" or of_sublayer) and (name != "router" or router_counts)]
    return dict(zip(names, torch.autograd.grad((y * dy).sum(), [at[name] for name in names])))


def fits(ours, exact, off, tokens):
    d = (ours.double() - exact).abs()
    print("largest error %.3g standard deviations, norm %.3g of theirs and %.3g of the gradient's" % (float((d / off).max()), float(d.norm() / off.norm()), float(d.norm() / exact.norm())), flush=True)
    return bool((d <= 10 * off).all()) and (tokens < 30 or bool(d.norm() <= 3 * off.norm()))


def check(got, weights, x, residual, experts, dy, dtype, of_sublayer):
    weights, x, residual, dy = {name: t.double() for name, t in weights.items()}, x.double(), residual.double(), dy.double()
    expected, numbers = exact(weights, x, residual, experts, dy, of_sublayer), followed(weights, x, residual, experts, dy, dtype, of_sublayer)
    for name, ours in got.items():
        print(name, end=": ")
        assert ours.shape == expected[name].shape and fits(ours, expected[name], numbers[name].off, len(x)), name


def inputs(T, E, k, hidden, inner, dtype, seed, device, norm=False):
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape, by=1.0):
        return (torch.randn(shape, device=device, generator=g) * by).to(dtype)

    x, residual, dy = normal(T, hidden), normal(T, hidden), normal(T, hidden)
    weights = {"norm": (1 + 0.1 * normal(hidden).float()).to(dtype), "router": normal(E, hidden, by=hidden ** -0.5), "gate": normal(E, inner, hidden, by=hidden ** -0.5),
               "up": normal(E, inner, hidden, by=hidden ** -0.5), "down": normal(E, hidden, inner, by=inner ** -0.5)}
    return weights, x, residual, dy


SIZES = [(1, 8, 2, 72, 40), (60, 6, 3, 72, 40), (700, 5, 2, 72, 40)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("of_sublayer", [False, True])
@pytest.mark.parametrize("T,E,k,hidden,inner", SIZES)
def test_mistakes_leave_the_bounds(T, E, k, hidden, inner, of_sublayer, dtype):
    """On the CPU: the numbers that are followed are autograd's, gradients rounded to their type stay inside the bounds, and gradients with something left out do not."""
    weights, x, residual, dy = inputs(T, E, k, hidden, inner, dtype, 3, "cpu")
    wide = {name: t.double() for name, t in weights.items()}
    args = x.double(), residual.double()
    total = args[0] + args[1]
    n = total * torch.rsqrt(total.square().mean(1, keepdim=True) + EPS) * wide["norm"] if of_sublayer else args[0]
    experts = torch.topk(n @ wide["router"].t(), k, 1).indices
    expected, numbers = exact(wide, *args, experts, dy.double(), of_sublayer), followed(wide, *args, experts, dy.double(), dtype, of_sublayer)
    for name, t in expected.items():
        assert torch.allclose(numbers[name].value, t, rtol=1e-9, atol=1e-9 * float(t.abs().max())), name
        assert fits(t.to(dtype), t, numbers[name].off, T), name

    def leaves(name, mistaken):
        return not fits(mistaken, expected[name], numbers[name].off, T)

    assert leaves("x", exact(wide, *args, experts, dy.double(), of_sublayer, router_counts=False)["x"])
    assert leaves("x", dy.double() if of_sublayer else torch.zeros_like(x.double()))
    for name in expected:
        assert leaves(name, torch.zeros_like(expected[name])) and leaves(name, 1.5 * expected[name]) and leaves(name, -expected[name]), name
    for name in ("gate", "up", "down", "router"):
        for e in experts.unique().tolist():
            t = expected[name].clone()
            t[e] = 0
            assert leaves(name, t), (name, e)
    if of_sublayer:
        assert leaves("x", expected["x"] - dy.double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,hidden,inner", [(1, 8, 2, 72, 40), (30, 6, 3, 72, 40), (60, 6, 3, 72, 40), (700, 5, 2, 72, 40), (300, 12, 3, 136, 72)])
def test_the_operators_one_after_the_other(T, E, k, hidden, inner, dtype):
    import test_expert_operators as experts_tests
    from tiramisu_amd import operators

    weights, x, residual, dy = inputs(T, E, k, hidden, inner, dtype, 5 + T, "cuda")
    chosen = operators.route(operators.linear(x, weights["router"]).y, k).experts.long()
    _, *got = experts_tests.sublayer(x, *[weights[name] for name in ("router", "gate", "up", "down")], k, dy)
    del weights["norm"]
    check(dict(zip(("x", "router", "gate", "up", "down"), got)), weights, x, residual, chosen, dy, dtype, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,hidden,inner", [(1, 8, 2, 72, 40), (60, 6, 3, 72, 40), (700, 5, 2, 72, 40), (300, 9, 3, 264, 120)])
def test_the_sublayer(T, E, k, hidden, inner, dtype):
    weights, x, residual, dy = inputs(T, E, k, hidden, inner, dtype, 7 + T, "cuda")
    layer = expert_feed_forward.ExpertFeedForward(hidden, inner, E, k, dtype=dtype)
    assert layer.eps == EPS and layer.activation == "silu"
    for name, t in weights.items():
        getattr(layer, name).copy_(t)
    _, kept = layer.forward(x, residual)
    dx, gradients = layer.backward(dy, kept)
    assert sorted(gradients) == sorted(layer.NAMES)
    check(dict(gradients, x=dx), weights, x, residual, kept.route.experts.long(), dy, dtype, True)


@pytest.mark.gpu
def test_a_step_of_training_moves_every_weight_by_its_gradient():
    def generator(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        return g

    teacher = expert_feed_forward.ExpertFeedForward(72, 40, 6, 2, generator=generator(11))
    layer, same = [expert_feed_forward.disturbed(teacher, 0.5, generator(13)) for _ in range(2)]
    rate, tokens = 0.1, 200
    g = generator(17)
    x, residual = [torch.randn((tokens, 72), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    expert_feed_forward.train(layer, teacher, 1, tokens, rate=rate, generator=generator(17))
    y, kept = same.forward(x, residual)
    _, gradients = same.backward(((y.float() - teacher.serve(x, residual).float()) * (2.0 / tokens)).to(torch.bfloat16), kept)
    for name in layer.NAMES:
        before = getattr(same, name)
        step = rate * (1 if name in ("norm", "router") else 6 / 2) * gradients[name].float()
        assert torch.equal(getattr(layer, name), (before.float() - step).to(torch.bfloat16)), name
        assert not torch.equal(getattr(layer, name), before), name
