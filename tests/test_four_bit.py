"""Weights in 4 bits (tiramisu_amd/operators.py: quantize_groups, four_bit_linear, four_bit_gated_linear) against their definitions in 64 bits; tolerances are those of test_operators.py."""
import math

import pytest
import torch

import test_operators as definitions
from tiramisu_amd import operators, runtime
from test_operators import HALVES, close, exact_activation, generator, normal, rounded, sum_error

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def widened(q, scale, columns):
    """The numbers that 4-bit rows stand for, in 64 bits"""
    codes = torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)[:, :columns].long()
    value = torch.tensor(VALUES + [-v for v in VALUES], device=q.device, dtype=torch.float64)[codes]
    power = torch.exp2(scale.double() - 127).masked_fill(scale == 255, math.nan)
    return value * power.repeat_interleave(32, 1)[:, :columns]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 31), (5, 32), (40, 97), (7, 1430), (300, 512)])
def test_quantize_groups(rows, columns, dtype):
    """Scale and values are exact: the smallest power of two that will do, the nearest value, ties to the even code."""
    x = normal((rows, columns), dtype, generator(rows + columns), 3.0)
    x[0, : columns // 2] = 0
    if rows > 2:
        x[1] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -5.0], device="cuda").repeat(columns)[:columns].to(dtype)      # ties
        x[2] *= 2.0 ** -12
    got = operators.quantize_groups(x)
    assert got.q.shape == (rows, (columns + 1) // 2) and got.scale.shape == (rows, (columns + 31) // 32)
    padded = torch.nn.functional.pad(x.double(), (0, -columns % 32)).view(rows, -1, 32)
    most = padded.abs().amax(2)
    exponent = torch.where(most > 0, torch.ceil(torch.log2(most.clamp(min=1e-300) / 6)), 0.0)
    assert torch.equal(got.scale.double(), exponent + 127)
    size = (padded.abs() * torch.exp2(-exponent)[..., None]).view(rows, -1)[:, :columns]
    table = torch.tensor(VALUES, device="cuda", dtype=torch.float64)
    off = (size[..., None] - table).abs()
    # (of two that are equally near the even one)
    code = (off + torch.tensor([0, 1e-9] * 4, device="cuda", dtype=torch.float64)).argmin(-1)
    ours = torch.stack((got.q & 15, got.q >> 4), -1).view(rows, -1)[:, :columns].long()
    assert torch.equal(ours & 7, code) and torch.equal((ours >> 3).bool(), torch.signbit(x))
    if columns % 2:
        assert not bool((got.q[:, -1] >> 4).any())


@pytest.mark.gpu
def test_quantize_groups_that_are_not_ordinary():
    """Numbers near the ends of 32 bits, and groups with an infinity or a NaN, whose scale is NaN; the other groups are as without."""
    x = torch.zeros((6, 64), device="cuda")
    x[0, 0], x[1, 3], x[2, 40], x[3, 5] = 3.4e38, 2.0 ** -149, math.nan, -math.inf
    x[2, 0] = 1.0
    q, scale = operators.quantize_groups(x)
    value = widened(q, scale, 64)
    assert [int(s) for s in scale[0]] == [127 + 126, 127] and 2.0 ** 127 <= float(value[0, 0]) <= 1.5 * 2.0 ** 128
    assert int(scale[1, 0]) == 0 and float(value[1, 3]) == 0
    assert int(scale[2, 1]) == 255 and int(scale[3, 0]) == 255 and int(scale[2, 0]) == 125 and float(value[2, 0]) == 1.0
    assert bool(torch.isnan(value[2, 32:]).all()) and bool(torch.isnan(value[3, :32]).all()) and not bool(value[4:].any())


PRODUCTS = [(1, 1, 1), (1, 17, 33), (3, 40, 8), (16, 16, 64), (17, 100, 72), (33, 24, 1000), (64, 130, 200), (65, 64, 64), (100, 70, 7), (128, 256, 128), (129, 130, 1001), (300, 1000, 520), (1, 300, 4100),
            (5, 33, 2048), (40, 50, 5000)]


def four_bit_inputs(M, N, K, dtype, seed, weights=1):
    g = generator(seed)
    x = normal((M, K), dtype, g)
    rows = [operators.quantize_groups(torch.randn((N, K), device="cuda", generator=g) * max(1, K) ** -0.5) for _ in range(weights)]
    return x, rows, x.double(), [widened(r.q, r.scale, K) for r in rows]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_four_bit_linear(M, N, K, dtype):
    x, (w,), xd, (wd,) = four_bit_inputs(M, N, K, dtype, M + N + K)
    g = generator(17)
    bias, residual = normal((N,), dtype, g), normal((M, N), dtype, g)
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    # float16 holds multiples of 2^-24: a weight of a small group may be off by half of that
    error = sum_error(K, size + bias.double().abs()) + (2.0 ** -25 * xd.abs().sum(1, keepdim=True) if dtype == torch.float16 else 0)
    for i, activation in enumerate(operators.ACTIVATIONS):
        b, r = bias if i != 1 else None, residual if i % 2 else None
        got = operators.four_bit_linear(x, w.q, w.scale, bias=b, residual=r, activation=activation)
        pre = z + (b.double() if b is not None else 0)
        y = exact_activation(activation, pre)
        if r is not None:
            y = y + r.double()
        close(got.y, y, rounded(y, 1.13 * error + 2.0 ** -22 * (pre.abs() + 1 + (0 if r is None else r.double().abs())), dtype), "%s y" % activation)
        assert torch.equal(got.y, operators.four_bit_linear(x, w.q, w.scale, bias=b, residual=r, activation=activation).y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_four_bit_gated_linear(M, N, K, dtype):
    x, (g, u), xd, (gd, ud) = four_bit_inputs(M, N, K, dtype, M + N + K, weights=2)
    gate, up = xd @ gd.t(), xd @ ud.t()
    lost = 2.0 ** -25 * xd.abs().sum(1, keepdim=True) if dtype == torch.float16 else 0
    eg, eu = [sum_error(K, xd.abs() @ w.abs().t()) + lost for w in (gd, ud)]
    for activation in ("silu", "gelu_tanh"):
        got = operators.four_bit_gated_linear(x, g.q, u.q, g.scale, u.scale, activation=activation)
        a = exact_activation(activation, gate)
        h = a * up
        close(got.h, h, rounded(h, (1.13 * eg + 2.0 ** -22 * (gate.abs() + 1)) * (up.abs() + eu) + a.abs() * eu + 2.0 ** -23 * h.abs(), dtype), "%s h" % activation)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 200])
def test_every_value_and_scale(M):
    """One row of weights for each value and scale: what a product with ones sums up, by exponents from 2^-126 to 2^125 in bfloat16."""
    q = torch.tensor([[c] + [0] * 15 for c in range(16)], device="cuda", dtype=torch.uint8).repeat(252, 1)
    scale = torch.arange(1, 253, device="cuda", dtype=torch.uint8).repeat_interleave(16)[:, None].contiguous()
    x = torch.ones((M, 32), device="cuda", dtype=torch.bfloat16)
    exact = widened(q, scale, 32)[:, 0].bfloat16()
    got = operators.four_bit_linear(x, q, scale).y
    normal_ones = exact.abs().float() >= 2.0 ** -126          # (the matrix instructions take numbers below as zero)
    assert torch.equal(got[:, normal_ones], exact[normal_ones].expand(M, -1))
    assert bool((got[:, ~normal_ones].float().abs() <= 2.0 ** -126).all())
    # a scale of NaN reaches its own outputs only
    scale[5] = 255
    again = operators.four_bit_linear(x, q, scale).y
    assert bool(torch.isnan(again[:, 5]).all()) and torch.equal(again[:, 6:], got[:, 6:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K,first", [(5, 33, 70, 0), (70, 66, 71, 1), (200, 140, 600, 3)])
def test_operands_within_larger_tensors(M, N, K, first, dtype):
    g = generator(43)

    def within(t, low, high):
        big = torch.full((t.shape[0] + 2, t.shape[1] + low + high), 255 if t.dtype == torch.uint8 else math.nan, device="cuda", dtype=t.dtype)
        big[1:-1, low:low + t.shape[1]] = t
        return big[1:-1, low:low + t.shape[1]]

    x, (a, b), _, _ = four_bit_inputs(M, N, K, dtype, 47, weights=2)
    r = normal((M, N), dtype, g)
    xv, qv, sv = within(x, first, 5), [within(t.q, first, 2) for t in (a, b)], [within(t.scale, first, 1) for t in (a, b)]
    assert torch.equal(operators.four_bit_linear(x, a.q, a.scale, residual=r).y, operators.four_bit_linear(xv, qv[0], sv[0], residual=within(r, first, 1)).y)
    assert torch.equal(operators.four_bit_gated_linear(x, a.q, b.q, a.scale, b.scale).h, operators.four_bit_gated_linear(xv, *qv, *sv).h)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [33, 97, 129, 255])
@pytest.mark.parametrize("M", [1, 40, 200])
def test_the_half_of_a_byte_behind_an_odd_row(M, K):
    """It is no weight, whatever it holds: with the row's last scale it would be infinity in float16."""
    x, (w,), _, _ = four_bit_inputs(M, 40, K, torch.float16, 59)
    last = w.q[:, K // 32 * 16:]
    last.zero_()
    w.scale[:, -1] = 127 + 30
    clean = operators.four_bit_linear(x, w.q, w.scale).y, operators.four_bit_gated_linear(x, w.q, w.q, w.scale, w.scale).h
    last[:, -1] = 0x70
    assert bool(torch.isfinite(clean[0]).all()) and torch.equal(operators.four_bit_linear(x, w.q, w.scale).y, clean[0])
    assert torch.equal(operators.four_bit_gated_linear(x, w.q, w.q, w.scale, w.scale).h, clean[1])


@pytest.mark.gpu
def test_infinities_reach_their_own_rows_only():
    for M in (3, 50, 200):
        x, (w,), _, _ = four_bit_inputs(M, 40, 100, torch.bfloat16, 53)
        clean = operators.four_bit_linear(x, w.q, w.scale).y
        x[1, 99], x[2, 0] = math.inf, math.nan
        got = operators.four_bit_linear(x, w.q, w.scale).y
        rows = [i for i in range(M) if i not in (1, 2)]
        assert torch.equal(got[rows], clean[rows]) and not bool(torch.isfinite(got[1:3]).any())


@pytest.mark.gpu
def test_more_tokens_than_parts_that_a_launch_has():
    """Four million tokens of a narrow product: the last are those of a call of their own."""
    M, N, K = 64 * 65535 + 65, 16, 64
    x, (w,), _, _ = four_bit_inputs(M, N, K, torch.bfloat16, 61)
    y = operators.four_bit_linear(x, w.q, w.scale).y
    xd, wd = x[-70:].double(), widened(w.q, w.scale, K)
    z = xd @ wd.t()
    close(y[-70:], z, rounded(z, sum_error(K, xd.abs() @ wd.abs().t()), torch.bfloat16), "y")


@pytest.mark.gpu
def test_no_tokens_and_no_terms():
    x, (w,), _, _ = four_bit_inputs(4, 40, 64, torch.bfloat16, 3)
    assert operators.four_bit_linear(x[:0], w.q, w.scale).y.shape == (0, 40) and operators.four_bit_gated_linear(x[:0], w.q, w.q, w.scale, w.scale).h.shape == (0, 40)
    bias = normal((40,), torch.bfloat16, generator(61))
    for M in (3, 200):
        none = torch.empty((M, 0), device="cuda", dtype=torch.bfloat16)
        assert torch.equal(operators.four_bit_linear(none, w.q[:, :0], w.scale[:, :0], bias=bias).y, bias.expand(M, 40))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 200])
def test_calls_in_a_graph(M):
    x, (a, b), _, _ = four_bit_inputs(M, 136, 264, torch.bfloat16, 3, weights=2)
    down = operators.quantize_groups(normal((264, 136), torch.float32, generator(4), 0.1))

    def layer():
        return operators.four_bit_linear(operators.four_bit_gated_linear(x, a.q, b.q, a.scale, b.scale).h, down.q, down.scale, residual=x).y

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = layer()
    for seed in range(3):
        x.copy_(normal(x.shape, torch.bfloat16, generator(seed)))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, layer())


def test_what_is_refused_without_a_gpu():
    x, q, s = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((8, 2), dtype=torch.uint8)
    for call in (lambda: operators.four_bit_linear(x, q, s), lambda: operators.four_bit_gated_linear(x, q, q, s, s), lambda: operators.quantize_groups(x)):
        with pytest.raises(ValueError, match="lives on cpu"):
            call()
    with pytest.raises(ValueError, match="x holds"):
        operators.four_bit_linear(x.float(), q, s)


@pytest.mark.gpu
def test_what_is_refused():
    x, q, s = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((8, 32), dtype=torch.uint8, device="cuda"), torch.zeros((8, 2), dtype=torch.uint8, device="cuda")
    refused = [
        (lambda: operators.four_bit_linear(x, q[:, :31], s), "weight"), (lambda: operators.four_bit_linear(x, q.int(), s), "weight holds"), (lambda: operators.four_bit_linear(x, q, s[:, :1]), "weight_scale"),
        (lambda: operators.four_bit_linear(x, q, s[:7]), "weight_scale"), (lambda: operators.four_bit_linear(x, q, s, bias=x[0, :7]), "bias"), (lambda: operators.four_bit_linear(x, q, s, residual=x), "residual"),
        (lambda: operators.four_bit_linear(x, q, s, activation="tanh"), "activation"), (lambda: operators.four_bit_gated_linear(x, q, q[:4], s, s), "up_weight"),
        (lambda: operators.four_bit_gated_linear(x, q, q, s, s[:4]), "up_scale"), (lambda: operators.quantize_groups(q), "x holds"), (lambda: operators.four_bit_linear(x.cpu(), q, s), "lives on cpu"),
    ]
    for call, message in refused:
        with pytest.raises(ValueError, match=message):
            call()


def test_what_the_c_abi_refuses(capfd):
    w, p = runtime.wrappers(), 4096
    calls = [w.tiramisu_hip_four_bit_linear(p, p, p, None, None, p, 4, 8, 1 << 22, 0, 0, 0, 0, 0, 2), w.tiramisu_hip_four_bit_linear(p, p, p, None, None, p, 4, 8, 64, 0, 0, 0, 0, 0, 3),
             w.tiramisu_hip_four_bit_linear(p, p, None, None, None, p, 4, 8, 64, 0, 0, 0, 0, 0, 2), w.tiramisu_hip_four_bit_linear(p, p, p, None, None, p, 4, 8, 64, 0, 0, 0, 0, 9, 2),
             w.tiramisu_hip_four_bit_gated_linear(p, p, None, p, p, p, 4, 8, 64, 0, 0, 0, 0, 0, 4, 2), w.tiramisu_hip_quantize_groups(p, p, None, 4, 8, 0, 2), w.tiramisu_hip_quantize_groups(p, p, p, 4, 8, 0, 3)]
    assert calls == [1] * len(calls)
    messages = capfd.readouterr().err.strip().splitlines()
    assert len(messages) == len(calls) and all(m.startswith("Error at tiramisu_hip_") for m in messages)


@pytest.mark.gpu
@pytest.mark.parametrize("M,times,K", [(1, 1, 32), (40, 1, 32), (200, 1, 32), (3001, 44, 1344)])
def test_the_least_and_the_largest_scales(M, times, K):
    """Exponents 0, 253 and 254 in bfloat16, through registers and through the widened copy: exact down to 2^-128, and infinite where the value is 2^128 or more."""
    for byte in (0, 253, 254):
        q = torch.zeros((16 * times, K // 2), device="cuda", dtype=torch.uint8)
        q[:, 0] = torch.arange(16, device="cuda", dtype=torch.uint8).repeat(times)
        scale = torch.full((16 * times, K // 32), byte, device="cuda", dtype=torch.uint8)
        exact = widened(q, scale, K)[:, 0]
        expected = torch.where(exact.abs() >= 2.0 ** 128, exact.sign() * math.inf, exact)
        got = operators.four_bit_linear(torch.ones((M, K), device="cuda", dtype=torch.bfloat16), q, scale).y
        print(byte, got[0, :16].tolist(), flush=True)
        assert torch.equal(got.double(), expected.nan_to_num(0, math.inf, -math.inf).expand(M, -1))


@pytest.mark.gpu
def test_groups_of_the_largest_numbers():
    """float32 numbers that the nearest values of their group bring to 2^128 keep their scale and value; in a product such a weight is infinite, as bfloat16 has no number there."""
    x = torch.zeros((2, 32), device="cuda")
    x[0, 0], x[1, 0] = 3.4e38, 2.0 ** 127
    r = operators.quantize_groups(x)
    assert [int(v) for v in r.scale[:, 0]] == [253, 252] and widened(r.q, r.scale, 32)[:, 0].tolist() == [2.0 ** 128, 2.0 ** 127]
    y = operators.four_bit_linear(torch.ones((1, 32), device="cuda", dtype=torch.bfloat16), r.q, r.scale).y
    assert y[0].tolist() == [math.inf, 2.0 ** 127]
