"""The operators of experts and of 4-bit weights together: a sublayer with experts trained and served from Python, one served in 4 bits, and both as compiled Tiramisu programs."""
import os
import subprocess

import pytest
import torch

from test_feed_forward import exact as exact_dense
from tiramisu_amd import build, expert_feed_forward, feed_forward, operators, runtime

PROGRAMS = os.path.join(build.PKG, "programs")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(shape, dtype, g):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def exact(layer, x, residual, experts):
    """In 64 bits, with the router's choice given; and the sum"""
    norm, router, gate, up, down = [getattr(layer, name).double() for name in layer.NAMES]
    s = x.double() + residual.double()
    n = s * torch.rsqrt(s.square().mean(1, keepdim=True) + layer.eps) * norm
    w = torch.softmax((n @ router.t()).gather(1, experts), 1)
    y = s
    for e in range(len(gate)):
        g = n @ gate[e].t()
        y = y + (w * (experts == e)).sum(1, keepdim=True) * ((g * torch.sigmoid(g) * (n @ up[e].t())) @ down[e].t())
    return y, s


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 200])
def test_forward(tokens):
    """Four results of the branch are rounded to bfloat16 on the way (norm, h, the experts' rows, and the logits, which are of order 1 and move each weight by as much of itself), each by 2^-8 of
    itself at most; and the sum and y by 2^-8 of themselves."""
    g = generator(3)
    layer = expert_feed_forward.ExpertFeedForward(264, 120, 9, 3, generator=g)
    x, r = [normal((tokens, 264), torch.bfloat16, g) for _ in range(2)]
    y, kept = layer.forward(x, r)
    ref, s = exact(layer, x, r, kept.route.experts.long())
    # (the logits: 2^-8 of up to 4, in two terms of the softmax)
    assert float((y.double() - ref).norm()) <= (3 + 2 * 4) * 2.0 ** -8 * float((ref - s).norm()) + 2 * 2.0 ** -8 * float(ref.norm())
    assert torch.equal(layer.serve(x, r), y) and kept.h.shape == (3 * tokens, 120)


@pytest.mark.gpu
def test_gradients_of_the_sublayer_against_differences():
    g = generator(7)
    layer = expert_feed_forward.ExpertFeedForward(72, 40, 5, 2, dtype=torch.float16, generator=g)
    x, r, dy = [normal((60, 72), torch.float16, g) for _ in range(3)]
    _, kept = layer.forward(x, r)
    experts = kept.route.experts.long()
    dx, gradients = layer.backward(dy, kept)
    for name, grad in [("x", dx)] + list(gradients.items()):
        at = x if name == "x" else getattr(layer, name)
        d = torch.randn(at.shape, device="cuda", generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = expert_feed_forward.ExpertFeedForward.__new__(expert_feed_forward.ExpertFeedForward)
            moved.eps = layer.eps
            for n in layer.NAMES:
                setattr(moved, n, getattr(layer, n).double() + (sign * 1e-6 * d if n == name else 0))
            ends.append(float((exact(moved, x.double() + (sign * 1e-6 * d if name == "x" else 0), r, experts)[0] * dy.double()).sum()))
        difference, ours = (ends[0] - ends[1]) / 2e-6, float((grad.double() * d).sum())
        # some twenty stored intermediates, each off by at most 2^-11 of itself
        bound = 24 * 2.0 ** -11 * float((grad.double().abs() * d.abs()).sum())
        print("%s: difference %.6g, gradient %.6g, bound %.3g" % (name, difference, ours, bound), flush=True)
        assert abs(difference - ours) <= bound, name


@pytest.mark.gpu
def test_training_runs_and_8_bits_follow():
    g = generator(5)
    teacher = expert_feed_forward.ExpertFeedForward(128, 64, 8, 2, generator=g)
    layer = expert_feed_forward.disturbed(teacher, 0.5, g)
    errors = expert_feed_forward.train(layer, teacher, 5, 256, generator=g)
    assert len(errors) == 5 and all(0 <= e < 1e3 for e in errors)
    x, r = [normal((64, 128), torch.bfloat16, g) for _ in range(2)]
    y, kept = layer.forward(x, r)
    small = layer.in_8_bits().serve(x, r)
    # e4m3 keeps 4 bits: each of five roundings (n, three matrices, h) is off by at most 2^-4 of itself, in rms by 2^-4 / sqrt 3 at most, independently
    assert float((small.double() - y.double()).norm()) <= (5 / 3) ** 0.5 * 2.0 ** -4 * float((y.double() - kept.sum.double()).norm()) + 2.0 ** -6 * float(y.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_4_bits_follow(tokens):
    """A value of e2m1 is off by at most half a step: 1/4 of the group's unit below 2, 1/2 to 4, 1 beyond, with the group's largest between 3 and 6 units, so by at most 1/3 of itself above 1/2 a unit and
    in rms by less than 0.15 of the group's rms; three matrices, independently, of which the branch is a product."""
    g = generator(9)
    layer = feed_forward.FeedForward(264, 600, generator=g)
    x, r = [normal((tokens, 264), torch.bfloat16, g) for _ in range(2)]
    y, s = exact_dense(layer, x, r)
    served = layer.in_4_bits().serve(x, r)
    assert float((served.double() - y).norm()) <= 3 ** 0.5 * 0.15 * float((y - s).norm()) + 2.0 ** -6 * float(y.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hidden,inner,experts,k", [(1, 1024, 512, 32, 4), (300, 520, 200, 6, 2)])
def test_tiramisu_program(tokens, hidden, inner, experts, k):
    """The compiled program's results are those of the same operators called one by one, bit for bit."""
    program = runtime.load(PROGRAMS, "expert_feed_forward_%dx%dx%dx%dx%d" % (tokens, hidden, inner, experts, k))
    g = generator(11)
    layer = expert_feed_forward.ExpertFeedForward(hidden, inner, experts, k, generator=g)
    s, y = [torch.empty((tokens, hidden), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for _ in range(2):
        x, r = [normal((tokens, hidden), torch.bfloat16, g) for _ in range(2)]
        program(x, r, layer.norm, layer.router, layer.gate, layer.up, layer.down, s, y)
        expected, kept = layer.forward(x, r)
        assert torch.equal(s, kept.sum) and torch.equal(y, expected)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hidden,inner", [(1, 1024, 4096), (300, 520, 1000)])
def test_tiramisu_program_in_4_bits(tokens, hidden, inner):
    program = runtime.load(PROGRAMS, "four_bit_feed_forward_%dx%dx%d" % (tokens, hidden, inner))
    g = generator(13)
    layer = feed_forward.FeedForward(hidden, inner, generator=g).in_4_bits()
    s, y = [torch.empty((tokens, hidden), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    x, r = [normal((tokens, hidden), torch.bfloat16, g) for _ in range(2)]
    program(x, r, layer.norm, layer.gate.q, layer.gate.scale, layer.up.q, layer.up.scale, layer.down.q, layer.down.scale, s, y)
    assert torch.equal(y, layer.serve(x, r)) and torch.equal(s, (x.float() + r.float()).bfloat16())


@pytest.mark.parametrize("call,message", [("hip_route(y, x, w, o, o, o, expr(4), expr(2), expr(1))", "holds"), ("hip_grouped_linear(x, y, x, y, expr(4), expr(4), expr(1), expr(2), expr(8))", "not int32"),
                                          ("hip_four_bit_linear(x, x, o, y, expr(4), expr(2), expr(8))", "not uint8"), ("hip_combine_rows(x, o, w, expr(4), expr(1), expr(4), expr(8))", "hold different types")])
def test_programs_say_what_does_not_fit(tmp_path, call, message):
    source = tmp_path / "wrong.cpp"
    source.write_text('''#include <tiramisu/tiramisu.h>
using namespace tiramisu;
int main() {
    tiramisu::init("wrong");
    buffer x("x", {4, 8}, p_bfloat16, a_input), w("w", {4, 8}, p_float32, a_output), o("o", {4, 1}, p_int32, a_input), y("y", {4, 2}, p_bfloat16, a_output);
    for (buffer *b : {&x, &w, &o, &y}) b->tag_gpu_global();
    computation c({var("once", 0, 1)}, %s);
    tiramisu::codegen({&x, &w, &o, &y}, "wrong.o", true);
}''' % call)
    subprocess.run(["g++", "-std=c++17", "-I" + build.INCLUDE, "-o", str(tmp_path / "gen"), str(source), "-L" + build.PKG, "-ltiramisu", "-Wl,-rpath," + build.PKG], check=True)
    r = subprocess.run([str(tmp_path / "gen")], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode != 0 and message in r.stdout + r.stderr, r.stdout + r.stderr
