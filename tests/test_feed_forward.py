"""The operators together: a feed-forward sublayer trained and served from Python, and the same forward pass as a compiled Tiramisu program."""
import os
import subprocess

import pytest
import torch

from tiramisu_amd import build, feed_forward, operators, runtime

PROGRAMS = os.path.join(build.PKG, "programs")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def exact(layer, x, residual):
    n = [t.double() for t in (layer.norm, layer.gate, layer.up, layer.down)]
    s = x.double() + residual.double()
    y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + layer.eps) * n[0]
    g = y @ n[1].t()
    return s + (g * torch.sigmoid(g) * (y @ n[2].t())) @ n[3].t(), s


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 40, 200])
def test_forward(tokens):
    """Four results are rounded to bfloat16 on the way (norm, h, and the sum, y): each is off by at most 2^-8 of itself, so the branch by some 3 x 2^-8
    of its norm, and y by 2^-8 of itself once more."""
    g = generator(3)
    layer = feed_forward.FeedForward(264, 600, generator=g)
    x, r = [torch.randn((tokens, 264), device="cuda", generator=g).bfloat16() for _ in range(2)]
    y, kept = layer.forward(x, r)
    ref, s = exact(layer, x, r)
    assert float((y.double() - ref).norm()) <= 3 * 2.0 ** -8 * float((ref - s).norm()) + 2 * 2.0 ** -8 * float(ref.norm())
    assert torch.equal(layer.serve(x, r), y) and kept.h.shape == (tokens, 600)


@pytest.mark.gpu
def test_training_learns_and_8_bits_follow():
    g = generator(5)
    teacher = feed_forward.FeedForward(128, 512, generator=g)
    layer = feed_forward.disturbed(teacher, 0.5, g)
    errors = feed_forward.train(layer, teacher, 60, 512, generator=g)
    assert errors[-1] < 0.4 * errors[0]         # (the same descent in 32 bits, by autograd and with another seed: 0.08 of the first error)
    small = layer.in_8_bits()
    x, r = [torch.randn((64, 128), device="cuda", generator=g).bfloat16() for _ in range(2)]
    y, s = exact(layer, x, r)
    # e4m3 keeps 4 bits: each of five roundings (n, three matrices, h) is off by at most 2^-4 of itself, in rms by 2^-4 / sqrt 3 at most, independently
    assert float((small.serve(x, r).double() - y).norm()) <= (5 / 3) ** 0.5 * 2.0 ** -4 * float((y - s).norm()) + 2.0 ** -7 * float(y.norm())


@pytest.mark.gpu
def test_gradients_of_the_sublayer_against_differences():
    g = generator(7)
    layer = feed_forward.FeedForward(72, 136, dtype=torch.float16, generator=g)
    x, r, dy = [torch.randn((24, 72), device="cuda", generator=g).half() for _ in range(3)]
    _, kept = layer.forward(x, r)
    dx, gradients = layer.backward(dy, kept)
    for name, grad in [("x", dx)] + list(gradients.items()):
        at = x if name == "x" else getattr(layer, name)
        d = torch.randn(at.shape, device="cuda", generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = feed_forward.FeedForward.__new__(feed_forward.FeedForward)
            moved.eps = layer.eps
            for n in layer.NAMES:
                setattr(moved, n, getattr(layer, n).double() + (sign * 1e-6 * d if n == name else 0))
            ends.append(float((exact(moved, x.double() + (sign * 1e-6 * d if name == "x" else 0), r)[0] * dy.double()).sum()))
        difference, ours = (ends[0] - ends[1]) / 2e-6, float((grad.double() * d).sum())
        # a dozen stored intermediates, each off by at most 2^-11 of itself
        assert abs(difference - ours) <= 16 * 2.0 ** -11 * float((grad.double().abs() * d.abs()).sum()), name


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hidden,inner", [(1, 1024, 4096), (300, 520, 1000), (2048, 1024, 4096)])
def test_tiramisu_program(tokens, hidden, inner):
    """The compiled program's results are those of the same operators called one by one, bit for bit."""
    program = runtime.load(PROGRAMS, "feed_forward_%dx%dx%d" % (tokens, hidden, inner))
    g = generator(11)
    layer = feed_forward.FeedForward(hidden, inner, generator=g)
    x, r = [torch.randn((tokens, hidden), device="cuda", generator=g).bfloat16() for _ in range(2)]
    s, y = torch.empty_like(x), torch.empty_like(x)
    for _ in range(2):
        program(x, r, layer.norm, layer.gate, layer.up, layer.down, s, y)
        expected, kept = layer.forward(x, r)
        assert torch.equal(s, kept.sum) and torch.equal(y, expected)


def test_programs_say_what_does_not_fit(tmp_path):
    """Buffers of different types are refused when the code is generated."""
    source = tmp_path / "wrong.cpp"
    source.write_text('''#include <tiramisu/tiramisu.h>
using namespace tiramisu;
int main() {
    tiramisu::init("wrong");
    buffer x("x", {4, 8}, p_bfloat16, a_input), w("w", {2, 8}, p_float32, a_input), y("y", {4, 2}, p_bfloat16, a_output);
    for (buffer *b : {&x, &w, &y}) b->tag_gpu_global();
    computation c({var("once", 0, 1)}, hip_linear(x, w, y, expr(4), expr(2), expr(8)));
    tiramisu::codegen({&x, &w, &y}, "wrong.o", true);
}''')
    subprocess.run(["g++", "-std=c++17", "-I" + build.INCLUDE, "-o", str(tmp_path / "gen"), str(source), "-L" + build.PKG, "-ltiramisu", "-Wl,-rpath," + build.PKG], check=True)
    r = subprocess.run([str(tmp_path / "gen")], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode != 0 and "hold different types" in r.stdout + r.stderr


def test_a_refused_call_in_a_program_ends_the_process():
    """(the reference's failure model) in a process of its own, without a GPU"""
    code = "from tiramisu_amd import runtime; w = runtime.wrappers(); w.tiramisu_hip_require(0); w.tiramisu_hip_require(w.tiramisu_hip_linear(1, 1, None, None, None, None, 1, None, 4, 4, 4, 0, 0, 0, 77, 2, 2))"
    r = subprocess.run(["python3", "-c", code], cwd=build.ROOT, capture_output=True, text=True)
    assert r.returncode == 1 and "activation 77" in r.stderr
    assert operators.ACTIVATIONS["silu"] == 4
