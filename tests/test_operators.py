"""The operators of a transformer's feed-forward sublayer (tiramisu_amd/operators.py) against their definitions in 64 bits.

Tolerances are derived, element by element.  With u the unit roundoff of a type (2^-24, 2^-11, 2^-8 for float32, float16, bfloat16), a
sum of n products whose magnitudes add up to S, formed in 32 bits in any order, is off by at most 2 (n + 8) 2^-24 S (the eight: scales, bias,
residual and the activation's few operations; the two: the matrix cores' own rounding of partial sums is not specified to the last bit);
rounding the result adds u |result|, and 2^-25 for float16's subnormal numbers.  Activations have slopes of at most 1.13.
The 8-bit matrix instructions of gfx950 add eight neighbouring products at a time, each cut off below 2^-12 of the largest one's power of two (seen
with pairs of products: 2^14 + 2^2 (1 + 1/8)^2 gives 2^14 + 4 within eight neighbours, and the exact sum across them): seven of eight may lose that much."""
import math

import pytest
import torch

from tiramisu_amd import operators, runtime

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
HALVES = [torch.bfloat16, torch.float16]
F8 = torch.float8_e4m3fn


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(shape, dtype, g, by=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * by).to(dtype)


def close(out, exact, bound, what):
    """|out - exact| <= bound, element by element, and finite where the exact value is."""
    d = (out.double() - exact).abs()
    worst = float((d / bound).max()) if out.numel() else 0.0
    print("%s: largest error is %.3g of its bound" % (what, worst), flush=True)
    assert out.shape == exact.shape and bool(torch.isfinite(out.double()).all()), what
    assert worst <= 1.0, what


def rounded(exact, error, dtype):
    """The bound of a result that is off by `error` ahead of its rounding to `dtype`."""
    return error + ROUNDOFF[dtype] * (exact.abs() + error) + LEAST[dtype]


def exact_activation(name, z):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def exact_slope(name, z):
    z = z.clone().requires_grad_()
    return torch.autograd.grad(exact_activation(name, z).sum(), z)[0]


# ---------------------------------------------------------------- norm

NORM_SHAPES = [(1, 1), (1, 7), (3, 64), (130, 100), (5, 513), (4, 1430), (2, 2049), (3, 4100), (2, 8200), (2, 16400), (3, 33001)]


def norm_inputs(rows, columns, dtype, seed, residual=True, by=1.0):
    g = generator(seed)
    x, r = normal((rows, columns), dtype, g, by), normal((rows, columns), dtype, g, by) if residual else None
    return x, r, (1 + normal((columns,), torch.float32, g, 0.1)).to(dtype)


def exact_norm(x, r, w, eps=1e-6):
    s = x.double() if r is None else x.double() + r.double()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, rstd, s * rstd * w.double()


def norm_error(columns, y):
    # squares, their sum and its root: (columns + 8) roundings, half of them through the root; the sum itself one more
    return (columns + 16) * 2.0 ** -24 * y.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", NORM_SHAPES)
def test_norm(rows, columns, dtype):
    for residual in (False, True):
        x, r, w = norm_inputs(rows, columns, dtype, 1 + columns, residual)
        s, rstd, y = exact_norm(x, r, w)
        got = operators.rms_norm(x, w, residual=r, keep_rstd=True)
        assert got.y.dtype == dtype and got.scale is None
        if residual:
            close(got.sum, s, rounded(s, 2.0 ** -24 * s.abs(), dtype), "sum")
        else:
            assert got.sum is x
        close(got.rstd[:, None], rstd, (columns + 16) * 2.0 ** -24 * rstd, "rstd")
        close(got.y, y, rounded(y, norm_error(columns, y) + 2.0 ** -24 * rstd * w.double().abs() * s.abs(), dtype), "y")


def nearest_e4m3(v):
    """What lies around a number of at most 448: half a step of e4m3."""
    e = torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -6)))
    return 2.0 ** (e - 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", NORM_SHAPES)
def test_norm_to_8_bits(rows, columns, dtype):
    x, r, w = norm_inputs(rows, columns, dtype, 2 + columns)
    s, rstd, y = exact_norm(x, r, w)
    got = operators.rms_norm(x, w, residual=r, eight_bit=True)
    assert got.y.dtype == F8 and got.scale.shape == (rows,)
    scale = y.abs().amax(1) / 448
    relative = (columns + 32) * 2.0 ** -24
    close(got.scale, scale, relative * scale, "scale")
    q = y / scale[:, None]
    close(got.y, q, nearest_e4m3(q) * (1 + 2.0 ** -10) + 2 * relative * q.abs(), "q")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 100), (40, 1430), (2, 40000)])
def test_quantize_rows(rows, columns, dtype):
    x = normal((rows, columns), dtype, generator(3), 3.0)
    x[0] = 0
    q, scale = operators.quantize_rows(x)
    assert float(scale[0]) == 1.0 and not bool(q[0].float().any())
    exact = x.double() / scale.double()[:, None]
    # (the quotient itself, rounded once: torch's division of a tensor by a number multiplies by the number's rounded reciprocal)
    assert torch.equal(scale[1:], (x[1:].double().abs().amax(1) / 448).float())
    close(q, exact, nearest_e4m3(exact) * (1 + 2.0 ** -10), "q")


@pytest.mark.gpu
def test_norm_of_rows_that_are_not_ordinary():
    """Rows of zeros, of the smallest and of very large numbers, with an infinity and with a NaN, among ordinary ones."""
    x, _, w = norm_inputs(8, 300, torch.float32, 5, residual=False)
    x[1], x[2], x[3] = 0, x[2] * 1e-30, x[3] * 1e15
    x[4, 17], x[5, 299] = math.inf, math.nan
    for eight_bit in (False, True):
        got = operators.rms_norm(x, w, eight_bit=eight_bit, keep_rstd=True)
        y = got.y.float() if got.scale is None else got.y.float() * got.scale[:, None]
        plain = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6) * w
        for row in (0, 1, 2, 3, 6, 7):
            assert torch.allclose(y[row], plain[row], rtol=0.07 if eight_bit else 1e-5, atol=float(plain[row].abs().max()) * 2 ** -9 if eight_bit else 0)
        assert not bool(torch.isfinite(y[4, 17])) and not bool(torch.isfinite(y[5, 299]))
    assert bool(torch.isnan(got.scale[4])) and bool(torch.isnan(got.scale[5])) and float(got.scale[1]) == 1.0


@pytest.mark.gpu
def test_norm_of_strided_rows():
    g = generator(7)
    for dtype in (torch.float32, torch.bfloat16):
        wide = normal((3, 5, 400), dtype, g)
        x, r = wide[..., 1:302], wide[..., 99:400]
        w = normal((301,), dtype, g)
        got, packed = operators.rms_norm(x, w, residual=r), operators.rms_norm(x.contiguous(), w, residual=r.contiguous())
        assert torch.equal(got.y, packed.y) and torch.equal(got.sum, packed.sum) and got.y.shape == (3, 5, 301)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 7), (700, 64), (1300, 100), (33, 513), (600, 1430), (9, 4100), (5, 8200), (2, 16400), (70, 33001)])
def test_norm_backward(rows, columns, dtype):
    g = generator(11)
    s, dy, ds = [normal((rows, columns), dtype, g) for _ in range(3)]
    w = (1 + normal((columns,), torch.float32, g, 0.1)).to(dtype)
    rstd = torch.rsqrt(s.float().square().mean(1) + 1e-6)
    for dsum in (None, ds):
        got = operators.rms_norm_backward(dy, s, w, rstd, dsum=dsum)
        xhat = s.double() * rstd.double()[:, None]
        gw = dy.double() * w.double()
        dx = rstd.double()[:, None] * (gw - xhat * (gw * xhat).mean(1, keepdim=True)) + (0 if dsum is None else ds.double())
        mean_size = (gw * xhat).abs().mean(1, keepdim=True)
        error = 2.0 ** -24 * (rstd.double()[:, None] * (8 * gw.abs() + (columns + 8) * xhat.abs() * mean_size) + 2 * ds.double().abs())
        close(got.dx, dx, rounded(dx, error, dtype), "dx")
        dw = (dy.double() * xhat).sum(0)
        close(got.dweight, dw, rounded(dw, (rows + 8) * 2.0 ** -24 * (dy.double() * xhat).abs().sum(0), dtype), "dweight")
        again = operators.rms_norm_backward(dy, s, w, rstd, dsum=dsum)
        assert torch.equal(again.dx, got.dx) and torch.equal(again.dweight, got.dweight)


@pytest.mark.gpu
def test_norm_backward_against_differences():
    """The gradients of a scalar against central differences of its 64-bit value along random directions."""
    g = generator(13)
    x, r, dy, ds = [normal((6, 130), torch.float32, g) for _ in range(4)]
    w = 1 + normal((130,), torch.float32, g, 0.1)
    kept = operators.rms_norm(x, w, residual=r, keep_rstd=True)
    got = operators.rms_norm_backward(dy, kept.sum, w, kept.rstd, dsum=ds)

    def value(x, w):
        s, _, y = exact_norm(x, r, w)
        return float((y * dy.double()).sum() + (s * ds.double()).sum())

    for grad, at, along in ((got.dx, 0, (6, 130)), (got.dweight, 1, (130,))):
        d = torch.randn(along, device="cuda", generator=g, dtype=torch.float64)
        h = 1e-5
        args = [[x.double() + (h * k * d if at == 0 else 0), w.double() + (h * k * d if at == 1 else 0)] for k in (1, -1)]
        difference = (value(*args[0]) - value(*args[1])) / (2 * h)
        # truncation h^2 of a third derivative of order 1 an element, rounding 2^-52 |value| / h, and 32-bit gradients: (130 + 16) 2^-24 an element
        bound = float((d.abs() * grad.double().abs()).sum()) * 150 * 2.0 ** -24 + 780 * (h * h * 50 + 2.0 ** -45 / h) + 1e-3
        assert abs(difference - float((grad.double() * d).sum())) <= bound


# ---------------------------------------------------------------- linear

def in_8_bits(t):
    scale = t.abs().amax(1) / 448
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (t / scale[:, None]).to(F8), scale


def product_inputs(M, N, K, dtype, seed, weights=1):
    """x, weights, their scales (None), and both in 64 bits."""
    g = generator(seed)
    x, ws = torch.randn((M, K), device="cuda", generator=g), [torch.randn((N, K), device="cuda", generator=g) * max(1, K) ** -0.5 for _ in range(weights)]
    if dtype != F8:
        x, ws = x.to(dtype), [w.to(dtype) for w in ws]
        return x, None, ws, [None] * weights, x.double(), [w.double() for w in ws]
    x, xs = in_8_bits(x)
    pairs = [in_8_bits(w) for w in ws]
    return x, xs, [q for q, _ in pairs], [s for _, s in pairs], x.double() * xs.double()[:, None], [q.double() * s.double()[:, None] for q, s in pairs]


def sum_error(n, size):
    return 2 * (n + 8) * 2.0 ** -24 * size


def cut_off(xd, wd, dtype):
    """What the 8-bit matrix instructions may cut off: 7 x 2^-12 of the largest of every eight neighbouring products."""
    if dtype != F8 or xd.shape[1] == 0:
        return 0.0
    pad = (0, -xd.shape[1] % 8)
    x, w = [torch.nn.functional.pad(t.abs(), pad).view(t.shape[0], -1, 8).float() for t in (xd, wd)]
    return torch.cat([(x[i:i + 8, None] * w[None]).amax(3).sum(2, dtype=torch.float64) for i in range(0, x.shape[0], 8)]) * (7 * 2.0 ** -12 * 1.001)


PRODUCTS = [(1, 1, 1), (1, 17, 33), (3, 40, 8), (16, 16, 64), (17, 100, 72), (33, 24, 1000), (64, 130, 200), (65, 64, 64), (66, 70, 7), (128, 256, 128),
            (200, 130, 1001), (257, 300, 129), (300, 1000, 520), (1030, 520, 300), (130, 260, 4100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(M, N, K, dtype):
    x, xs, (w,), (ws,), xd, (wd,) = product_inputs(M, N, K, dtype, M + N + K)
    g = generator(17)
    out = torch.float16 if dtype == torch.float16 else torch.bfloat16
    bias, residual = normal((N,), out, g), normal((M, N), out, g)
    z, size, cut = xd @ wd.t(), xd.abs() @ wd.abs().t(), cut_off(xd, wd, dtype)
    for i, activation in enumerate(operators.ACTIVATIONS):
        b, r, keep = (bias if i != 1 else None), (residual if i % 2 else None), i >= 3
        got = operators.linear(x, w, bias=b, residual=r, activation=activation, x_scale=xs, weight_scale=ws, keep_pre=keep)
        pre = z + (b.double() if b is not None else 0)
        error = sum_error(K, size + bias.double().abs()) + cut
        y = exact_activation(activation, pre)
        if r is not None:
            y = y + r.double()
        close(got.y, y, rounded(y, 1.13 * error + 2.0 ** -22 * (pre.abs() + 1 + (0 if r is None else r.double().abs())), out), "%s y" % activation)
        assert (got.pre is not None) == keep
        if keep:
            close(got.pre, pre, rounded(pre, error, out), "%s pre" % activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_gated_linear(M, N, K, dtype):
    x, xs, ws, scales, xd, (gd, ud) = product_inputs(M, N, K, dtype, M + N + K, weights=2)
    gate, up = xd @ gd.t(), xd @ ud.t()
    sizes = xd.abs() @ gd.abs().t(), xd.abs() @ ud.abs().t()
    cuts = cut_off(xd, gd, dtype), cut_off(xd, ud, dtype)
    out = torch.float16 if dtype == torch.float16 else torch.bfloat16
    for i, activation in enumerate(operators.ACTIVATIONS):
        keep = i % 2 == 0
        got = operators.gated_linear(x, ws[0], ws[1], activation=activation, x_scale=xs, gate_scale=scales[0], up_scale=scales[1], keep_pre=keep)
        a = exact_activation(activation, gate)
        h = a * up
        eg, eu = [sum_error(K, s) + c for s, c in zip(sizes, cuts)]
        ea = 1.13 * eg + 2.0 ** -22 * (gate.abs() + 1)
        close(got.h, h, rounded(h, ea * (up.abs() + eu) + a.abs() * eu + 2.0 ** -23 * h.abs(), out), "%s h" % activation)
        if keep:
            close(got.gate, gate, rounded(gate, eg, out), "gate")
            close(got.up, up, rounded(up, eu, out), "up")


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(2, 3, 4), (70, 80, 90)])
def test_8_bit_results_in_float16(M, N, K):
    x, xs, ws, scales, xd, (gd, ud) = product_inputs(M, N, K, F8, 3, weights=2)
    got = operators.linear(x, ws[0], x_scale=xs, weight_scale=scales[0], dtype=torch.float16)
    y = xd @ gd.t()
    close(got.y, y, rounded(y, sum_error(K, xd.abs() @ gd.abs().t()) + cut_off(xd, gd, F8), torch.float16), "y")
    assert operators.gated_linear(x, ws[0], ws[1], x_scale=xs, gate_scale=scales[0], up_scale=scales[1], dtype=torch.float16).h.dtype == torch.float16


BACKWARD = [(1, 1, 1), (3, 5, 2), (64, 64, 64), (70, 33, 129), (257, 130, 70), (500, 64, 320), (1500, 130, 258), (300, 1000, 65)]


def backward_bound(dtype, exact, terms, sizes):
    """A product over `terms` of factors, of which one was rounded to `dtype` ahead of it: sizes, the sum of the products' magnitudes."""
    return rounded(exact, (ROUNDOFF[dtype] * 1.01 + 2 * (terms + 16) * 2.0 ** -24) * sizes + terms * LEAST[dtype] * 8, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", BACKWARD)
def test_linear_backward(M, N, K, dtype):
    x, _, (w,), _, xd, (wd,) = product_inputs(M, N, K, dtype, 23 + M)
    g = generator(29)
    dy, pre = normal((M, N), dtype, g), normal((M, N), dtype, g, 2.0)
    for i, activation in enumerate(operators.ACTIVATIONS):
        p = None if activation == "none" else pre
        got = operators.linear_backward(dy, x, w, pre=p, activation=activation, bias=i % 2 == 0)
        dz = dy.double() if p is None else dy.double() * exact_slope(activation, pre.double())
        # the slope of an activation is of order 1: its 32-bit operations' error is an absolute one, 16 roundings
        slack = 16 * 2.0 ** -24 * dy.double().abs()
        size = dz.abs() + slack / ROUNDOFF[dtype]
        close(got.dx, dz @ wd, backward_bound(dtype, dz @ wd, N, size @ wd.abs()), "%s dx" % activation)
        close(got.dweight, dz.t() @ xd, backward_bound(dtype, dz.t() @ xd, M, size.t() @ xd.abs()), "%s dweight" % activation)
        assert (got.dbias is not None) == (i % 2 == 0)
        if got.dbias is not None:
            close(got.dbias, dz.sum(0), rounded(dz.sum(0), (2 * (M + 8) * 2.0 ** -24 * dz.abs() + slack).sum(0), dtype), "%s dbias" % activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", BACKWARD)
def test_gated_linear_backward(M, N, K, dtype):
    x, _, (wg, wu), _, xd, (gd, ud) = product_inputs(M, N, K, dtype, 31 + M, weights=2)
    g = generator(37)
    dh, gate, up = normal((M, N), dtype, g), normal((M, N), dtype, g, 2.0), normal((M, N), dtype, g)
    for activation in operators.ACTIVATIONS:
        got = operators.gated_linear_backward(dh, x, wg, wu, gate, up, activation=activation)
        zd = gate.double()
        dgate, dup = dh.double() * up.double() * exact_slope(activation, zd), dh.double() * exact_activation(activation, zd)
        slack = 16 * 2.0 ** -24 * dh.double().abs() * (1 + up.double().abs() + zd.abs()) / ROUNDOFF[dtype]
        sg, su = dgate.abs() + slack, dup.abs() + slack
        dx = dgate @ gd + dup @ ud
        close(got.dx, dx, backward_bound(dtype, dx, 2 * N, sg @ gd.abs() + su @ ud.abs()), "%s dx" % activation)
        close(got.dgate_weight, dgate.t() @ xd, backward_bound(dtype, dgate.t() @ xd, M, sg.t() @ xd.abs()), "%s dgate_weight" % activation)
        close(got.dup_weight, dup.t() @ xd, backward_bound(dtype, dup.t() @ xd, M, su.t() @ xd.abs()), "%s dup_weight" % activation)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Along random directions: central differences of the 64-bit value of the whole sublayer's products against the operators' gradients."""
    M, N, K = 24, 40, 56
    g = generator(41)
    x, wg, wu = normal((M, K), torch.float16, g), normal((N, K), torch.float16, g, 0.15), normal((N, K), torch.float16, g, 0.15)
    w, b, dy = normal((K, N), torch.float16, g, 0.15), normal((K,), torch.float16, g), normal((M, K), torch.float16, g)
    gated = operators.gated_linear(x, wg, wu, keep_pre=True)
    out = operators.linear(gated.h, w, bias=b, activation="gelu", keep_pre=True)
    back = operators.linear_backward(dy, gated.h, w, pre=out.pre, activation="gelu", bias=True)
    first = operators.gated_linear_backward(back.dx, x, wg, wu, gated.gate, gated.up)

    def value(x, wg, wu, w, b):
        h = exact_activation("silu", x @ wg.t()) * (x @ wu.t())
        return (exact_activation("gelu", h @ w.t() + b) * dy.double()).sum()

    at = [t.double() for t in (x, wg, wu, w, b)]
    grads = (first.dx, first.dgate_weight, first.dup_weight, back.dweight, back.dbias)
    for i, grad in enumerate(grads):
        d = torch.randn(grad.shape, device="cuda", generator=g, dtype=torch.float64)
        ends = [value(*[t + (k * 1e-6 * d if j == i else 0) for j, t in enumerate(at)]) for k in (1, -1)]
        difference = float(ends[0] - ends[1]) / 2e-6
        # every stored intermediate (gate, up, h, pre, dz, dh, dgate, dup, the gradient) is off by at most 2^-11 of itself: taken together sixteen
        # times that of the sum of magnitudes
        bound = 16 * 2.0 ** -11 * float((grad.double().abs() * d.abs()).sum())
        print("difference %.6g, gradient %.6g, bound %.3g" % (difference, float((grad.double() * d).sum()), bound))
        assert abs(difference - float((grad.double() * d).sum())) <= bound


# ---------------------------------------------------------------- memory, strides, streams

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("M,N,K,first", [(5, 33, 70, 0), (70, 66, 71, 1), (130, 140, 200, 3), (300, 260, 100, 2)])
def test_operands_within_larger_tensors(M, N, K, first, dtype):
    """Rows that go on into infinities and NaN, that begin at odd elements and are odd strides apart: neighbours do not count, and results
    are those of dense operands."""
    g = generator(43)

    def within(t, low, high):
        big = torch.full((t.shape[0] + 2, t.shape[1] + low + high), math.nan, device="cuda").to(t.dtype)
        if t.dtype != F8:
            big[1::2] = math.inf
        big[1:-1, low:low + t.shape[1]] = t
        return big[1:-1, low:low + t.shape[1]]

    x, xs, ws, scales, _, _ = product_inputs(M, N, K, dtype, 47, weights=2)
    xv, wv = within(x, first, 5), [within(w, first, 2) for w in ws]
    out = torch.float16 if dtype == torch.float16 else torch.bfloat16
    r = normal((M, N), out, g)
    a = operators.linear(x, ws[0], residual=r, x_scale=xs, weight_scale=scales[0])
    b = operators.linear(xv, wv[0], residual=within(r, first, 1), x_scale=xs, weight_scale=scales[0])
    assert torch.equal(a.y, b.y)
    a = operators.gated_linear(x, ws[0], ws[1], x_scale=xs, gate_scale=scales[0], up_scale=scales[1])
    b = operators.gated_linear(xv, wv[0], wv[1], x_scale=xs, gate_scale=scales[0], up_scale=scales[1])
    assert torch.equal(a.h, b.h)
    if dtype == F8:
        return
    dy, pre, up = [normal((M, N), dtype, g) for _ in range(3)]
    dyv, prev, upv = [within(t, first, 2) for t in (dy, pre, up)]
    for activation in ("none", "silu"):
        p, pv = (None, None) if activation == "none" else (pre, prev)
        a, b = operators.linear_backward(dy, x, ws[0], pre=p, activation=activation, bias=True), operators.linear_backward(dyv, xv, wv[0], pre=pv, activation=activation, bias=True)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    a, b = operators.gated_linear_backward(dy, x, ws[0], ws[1], pre, up), operators.gated_linear_backward(dyv, xv, wv[0], wv[1], prev, upv)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_infinities_reach_their_own_rows_and_columns_only():
    for M, N, K in ((3, 40, 100), (130, 140, 100)):
        x, _, (w, v), _, _, _ = product_inputs(M, N, K, torch.bfloat16, 53, weights=2)
        clean, clean_h = operators.linear(x, w).y, operators.gated_linear(x, w, v).h
        x[1, K - 1], w[5, 0] = math.inf, math.nan
        for got, was in ((operators.linear(x, w).y, clean), (operators.gated_linear(x, w, v).h, clean_h)):
            rows, columns = [i for i in range(M) if i != 1], [j for j in range(N) if j != 5]
            assert torch.equal(got[rows][:, columns], was[rows][:, columns])
            assert not bool(torch.isfinite(got[1]).any()) and bool(torch.isnan(got[:, 5]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [7, 300, 40000])
def test_rows_of_the_smallest_numbers_to_8_bits(columns):
    """Numbers below half of 448 times the smallest one have a scale of zero in 32 bits: such rows become zeros with scale 1, not NaN.  Somewhat larger ones keep a scale of few bits."""
    least = 2.0 ** -149
    x = torch.zeros((5, columns), device="cuda")
    x[0, 1], x[1, ::2], x[2, 3], x[3, :], x[4, 2] = least, 100 * least, 223 * least, 400 * least, -1e-40
    q, scale = operators.quantize_rows(x)
    assert [float(s) / least for s in scale[3:4]] == [1.0] and bool((scale[:3] == 1).all())
    values = q.float().double() * scale.double()[:, None]
    assert bool(torch.isfinite(values).all()) and not bool(values[:3].any()) and torch.equal(values == 0, (x == 0) | (scale[:, None] == 1))
    # (400: between 384 and 416 in e4m3; 1e-40: within half a step of its 4 bits, and half a unit of the scale's 8)
    assert bool(((values[3] - 400 * least).abs() <= 16 * least).all()) and abs(float(values[4, 2]) + 1e-40) <= 1e-40 * (2.0 ** -4 + 2.0 ** -7)
    w = torch.ones(columns, device="cuda")
    got = operators.rms_norm(x, w, eps=1.0, eight_bit=True)
    assert torch.equal(got.y.float(), q.float()) and torch.equal(got.scale, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_of_rows_without_elements(dtype):
    """Their scale is that of a row of zeros, their length is NaN like the mean of nothing: what is returned is written, whatever the memory held."""
    stale = [torch.full((5,), 7.0, device="cuda") for _ in range(8)]
    del stale                                  # (what the results' memory held)
    x, w = torch.empty((5, 0), dtype=dtype, device="cuda"), torch.empty((0,), dtype=dtype, device="cuda")
    q = operators.quantize_rows(x)
    assert q.q.shape == (5, 0) and bool((q.scale == 1).all())
    for residual in (None, x):
        got = operators.rms_norm(x, w, residual=residual, eight_bit=True, keep_rstd=True)
        assert got.y.shape == got.sum.shape == (5, 0) and bool((got.scale == 1).all()) and bool(torch.isnan(got.rstd).all())
    assert bool(torch.isnan(operators.rms_norm(x.view(5, 1, 0), w, keep_rstd=True).rstd).all())
    back = operators.rms_norm_backward(x, x, w, got.rstd)
    assert back.dx.shape == (5, 0) and back.dweight.shape == (0,)
    with pytest.raises(ValueError, match="rstd"):
        operators.rms_norm_backward(x, x, w, got.rstd[:0])


@pytest.mark.gpu
@pytest.mark.parametrize("activation", list(operators.ACTIVATIONS))
@pytest.mark.parametrize("M,N,K", [(3, 40, 100), (130, 140, 100), (100, 64, 4100)])
def test_activation_of_an_infinite_sum(M, N, K, activation):
    """Every activation of plus infinity is that: few tokens, tiles, and sums that were split; the other rows are what they are without it."""
    g = generator(101)
    x, w, up = [normal(shape, torch.bfloat16, g).abs() for shape in ((M, K), (N, K), (N, K))]
    clean = operators.linear(x, w, activation=activation).y
    x[1, K // 2] = math.inf
    got, h = operators.linear(x, w, activation=activation, keep_pre=True), operators.gated_linear(x, w, up, activation=activation).h
    rows = [i for i in range(M) if i != 1]
    assert bool((got.pre[1] == math.inf).all()) and bool((got.y[1] == math.inf).all()) and bool((h[1] == math.inf).all())
    assert torch.equal(got.y[rows], clean[rows])


@pytest.mark.gpu
def test_no_tokens_and_no_terms():
    x = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    w = normal((40, 64), torch.bfloat16, generator(59))
    assert operators.linear(x, w).y.shape == (0, 40) and operators.gated_linear(x, w, w).h.shape == (0, 40)
    assert operators.rms_norm(x, w[0]).y.shape == (0, 64)
    got = operators.linear_backward(torch.empty((0, 40), device="cuda", dtype=torch.bfloat16), x, w, bias=True)
    assert not bool(got.dweight.any()) and not bool(got.dbias.any()) and got.dx.shape == (0, 64)
    e = torch.empty((0, 40), device="cuda", dtype=torch.bfloat16)
    got = operators.gated_linear_backward(e, x, w, w, e, e)
    assert not bool(got.dgate_weight.any()) and not bool(got.dup_weight.any())
    got = operators.rms_norm_backward(x, x, w[0], torch.empty(0, device="cuda"))
    assert not bool(got.dweight.any())
    # no terms: what is left is the bias
    for M in (3, 100):
        none = torch.empty((M, 0), device="cuda", dtype=torch.bfloat16)
        b = normal((40,), torch.bfloat16, generator(61))
        assert torch.equal(operators.linear(none, torch.empty((40, 0), device="cuda", dtype=torch.bfloat16), bias=b).y, b.expand(M, 40))


@pytest.mark.gpu
def test_operands_beyond_4_gib():
    """Rows a long way apart: the last of them begin behind 2^32 bytes, in the operand of a forward product, and in that of a weight's gradient, whose
    k runs down the columns."""
    M, N, K, step = 2400, 72, 80, 1 << 20
    g = generator(67)
    far = torch.empty(M * step, dtype=torch.bfloat16, device="cuda").view(M, step)[:, :K]
    x = normal((M, K), torch.bfloat16, g)
    far.copy_(x)
    w, dy = normal((N, K), torch.bfloat16, g, 0.1), normal((M, N), torch.bfloat16, g)
    assert torch.equal(operators.linear(far, w).y, operators.linear(x, w).y)
    assert torch.equal(operators.linear(far[-5:], w).y, operators.linear(x[-5:], w).y)
    assert torch.equal(operators.linear_backward(dy, far, w).dweight, operators.linear_backward(dy, x, w).dweight)
    assert torch.equal(operators.rms_norm(far, w[0]).y, operators.rms_norm(x, w[0]).y)


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
def test_calls_follow_torchs_work_on_their_stream(side):
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    g = generator(71)
    w, x0 = normal((300, 1000), torch.bfloat16, g, 0.05), normal((100, 1000), torch.bfloat16, g)
    expected = operators.linear(x0 * 2, w, activation="silu").y.float() + 1
    torch.cuda.synchronize()
    a = torch.randn((6000, 6000), device="cuda")
    with torch.cuda.stream(stream):
        for _ in range(3):
            a = a @ a * 1e-4                       # keeps the stream busy for some ms
        x = x0 * 2
        y = operators.linear(x, w, activation="silu").y
        x.zero_()                                  # behind the call: must not reach it
        got = y.float() + 1
    torch.cuda.synchronize()
    assert torch.equal(got, expected)


@pytest.mark.gpu
def test_calls_in_a_graph():
    """The sublayer recorded once and replayed on new inputs, with eager work between the replays."""
    g = generator(73)
    x, r = normal((70, 1001), torch.bfloat16, g), normal((70, 1001), torch.bfloat16, g)
    w, wg, wu, wd = 1 + normal((1001,), torch.bfloat16, g, 0.1), *[normal(s, torch.bfloat16, g, 0.03) for s in ((400, 1001), (400, 1001), (1001, 400))]

    def sublayer():
        n = operators.rms_norm(x, w, residual=r, keep_rstd=True)
        h = operators.gated_linear(n.y, wg, wu, keep_pre=True)
        out = operators.linear(h.h, wd, residual=n.sum).y
        d = operators.linear_backward(out, h.h, wd)
        e = operators.gated_linear_backward(d.dx, n.y, wg, wu, h.gate, h.up)
        f = operators.rms_norm_backward(e.dx, n.sum, w, n.rstd, dsum=out)
        return out, d.dweight, e.dgate_weight, e.dup_weight, f.dx, f.dweight

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            sublayer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = sublayer()
    for seed in range(3):
        x.copy_(normal((70, 1001), torch.bfloat16, generator(seed)))
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        for u, v in zip(got, sublayer()):
            assert torch.equal(u, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("M,N,K", [(1030, 1990, 130), (1500, 1000, 77), (960, 1700, 512)])
def test_linear_of_some_two_hundred_tiles(M, N, K, dtype):
    test_linear(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", [(1030, 130, 990), (1000, 700, 500), (77, 1100, 1500)])
def test_linear_backward_of_some_two_hundred_tiles(M, N, K, dtype):
    test_linear_backward(M, N, K, dtype)


@pytest.mark.gpu
def test_a_graph_recorded_without_a_call_before():
    """Scratch (the activation's gradient, rows that are moved, sums of columns) is allocated while the stream records."""
    g = generator(89)
    x, w, dy, pre = normal((301, 77), torch.bfloat16, g), normal((95, 77), torch.bfloat16, g), normal((301, 95), torch.bfloat16, g), normal((301, 95), torch.bfloat16, g)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = operators.linear_backward(dy, x, w, pre=pre, activation="gelu", bias=True)
    for seed in range(3):
        dy.copy_(normal((301, 95), torch.bfloat16, generator(seed)))
        graph.replay()
        replayed = [t.clone() for t in got]
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(replayed, operators.linear_backward(dy, x, w, pre=pre, activation="gelu", bias=True)))


@pytest.mark.gpu
def test_more_rows_than_a_launch_holds():
    """The last of 2^22 + 77 rows are those of a call of their own."""
    rows = (1 << 22) + 77
    x = normal((rows, 8), torch.bfloat16, generator(97))
    w = x[0]
    got, last = operators.rms_norm(x, w, residual=x, eight_bit=True), operators.rms_norm(x[-200:], w, residual=x[-200:], eight_bit=True)
    assert torch.equal(got.y[-200:].float(), last.y.float()) and torch.equal(got.scale[-200:], last.scale) and torch.equal(got.sum[-200:], last.sum)
    kept = operators.rms_norm(x, w, keep_rstd=True)
    assert torch.equal(kept.rstd[-200:], operators.rms_norm(x[-200:], w, keep_rstd=True).rstd)


@pytest.mark.gpu
def test_launches_are_recorded_by_the_profile():
    x, w = normal((4, 64), torch.bfloat16, generator(79)), normal((64, 64), torch.bfloat16, generator(83))
    records = runtime.profile(lambda: (operators.rms_norm(x, w[0]), operators.linear(x, w), operators.gated_linear(x, w, w)))
    assert [name for name, _ in records] == ["tiramisu_hip_rms_norm", "tiramisu_hip_linear", "tiramisu_hip_gated_linear"]
    assert all(ms > 0 for _, ms in records)


# ---------------------------------------------------------------- refusals

def test_what_is_refused_without_a_gpu():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((8, 64), dtype=torch.bfloat16)
    for call in (lambda: operators.rms_norm(x, w[0]), lambda: operators.linear(x, w), lambda: operators.gated_linear(x, w, w), lambda: operators.quantize_rows(x)):
        with pytest.raises(ValueError, match="lives on cpu"):
            call()
    with pytest.raises(ValueError, match="holds torch.int32"):
        operators.rms_norm(x.int(), w[0])
    with pytest.raises(ValueError, match="holds torch.float32"):
        operators.linear(x.float(), w.float())
    with pytest.raises(ValueError, match="x is a tensor"):
        operators.linear([1.0], w)


@pytest.mark.gpu
def test_gradients_are_not_dropped_silently():
    """A tensor that requires a gradient is refused while gradients are recorded, in any place; otherwise it is a tensor like others."""
    g = generator(103)
    x, w, h = normal((4, 64), torch.bfloat16, g), normal((8, 64), torch.bfloat16, g), normal((4, 8), torch.bfloat16, g)
    p, rstd = torch.nn.Parameter(w), torch.ones(4, device="cuda")
    calls = [lambda w: operators.linear(x, w).y, lambda w: operators.gated_linear(x, w, w).h, lambda w: operators.rms_norm(x, w[0]).y, lambda w: operators.quantize_rows(w).scale,
             lambda w: operators.linear(x, p.detach(), residual=h, bias=w[:, 0].contiguous()).y, lambda w: operators.rms_norm(x, p.detach()[0], residual=w[:4]).sum,
             lambda w: operators.linear_backward(h, x, w).dx, lambda w: operators.rms_norm_backward(x, x, w[0], rstd).dx]
    for call in calls:
        with pytest.raises(ValueError, match="requires a gradient"):
            call(p)
        plain = call(w)
        for without in (torch.no_grad(), torch.inference_mode()):
            with without:
                assert torch.equal(call(p), plain)
        assert not plain.requires_grad


@pytest.mark.gpu
def test_what_is_refused():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((8, 64), dtype=torch.bfloat16, device="cuda")
    h = torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda")
    x8, w8, one = x.to(F8), w.to(F8), torch.ones(4, device="cuda")
    refused = [
        (lambda: operators.linear(x, w[:, :32]), "weight"), (lambda: operators.linear(x, w.half()), "weight holds"), (lambda: operators.linear(x, w[0]), "weight"),
        (lambda: operators.linear(x, w, bias=torch.zeros(9, dtype=torch.bfloat16, device="cuda")), "bias"),
        (lambda: operators.linear(x, w, bias=torch.zeros(8, device="cuda")), "bias"), (lambda: operators.linear(x, w, residual=x), "residual has shape"),
        (lambda: operators.linear(x, w, activation="tanh"), "activation"), (lambda: operators.linear(x, w, x_scale=one), "scales belong"),
        (lambda: operators.linear(x8, w8), "scales belong"), (lambda: operators.linear(x8, w8, x_scale=one, weight_scale=one), "weight_scale"),
        (lambda: operators.linear(x, w, dtype=torch.float16), "results"), (lambda: operators.linear(x.t(), w[:, :4]), "next to each other"),
        (lambda: operators.linear(x[:1].expand(4, 64), w), "overlap"), (lambda: operators.linear(torch.zeros((3, 4, 2, 64), dtype=torch.bfloat16, device="cuda")[:, ::2], w), "one stride"),
        (lambda: operators.gated_linear(x, w, w[:4]), "up_weight"), (lambda: operators.gated_linear(x8, w8, w8, x_scale=one, gate_scale=torch.ones(8, device="cuda")), "up_scale"),
        (lambda: operators.rms_norm(x, w[0][:32]), "weight"), (lambda: operators.rms_norm(x, w[0].float()), "weight"), (lambda: operators.rms_norm(x, w[0], residual=h), "residual"),
        (lambda: operators.rms_norm_backward(h, x, w[0], one), "dy"), (lambda: operators.rms_norm_backward(x, x, w[0], one[:3]), "rstd"),
        (lambda: operators.linear_backward(h, x, w, activation="relu"), "pre"), (lambda: operators.linear_backward(h, x, w, pre=h), "pre"),
        (lambda: operators.linear_backward(x, x, w), "dy has shape"), (lambda: operators.gated_linear_backward(h, x, w, w, h, x), "up has shape"),
    ]
    for call, message in refused:
        with pytest.raises(ValueError, match=message):
            call()


def test_what_the_c_abi_refuses(capfd):
    """A message on stderr, 1, and nothing launched: the calls return before they reach the device (addresses here are no memory)."""
    w = runtime.wrappers()
    p, far = 4096, 1 << 32
    assert w.tiramisu_hip_rms_norm(p, None, p, p, None, None, None, far, 8, 0, 0, 1e-6, 2, 2) == 1
    assert w.tiramisu_hip_rms_norm(p, None, p, p, None, None, None, 4, 8, 0, 0, 1e-6, 3, 3) == 1
    assert w.tiramisu_hip_rms_norm(p, None, p, p, None, None, None, 4, 8, 0, 0, 1e-6, 2, 3) == 1       # 8 bits without scales
    assert w.tiramisu_hip_rms_norm(p, p, p, p, None, None, None, 4, 8, 0, 0, 1e-6, 2, 2) == 1          # a residual without a sum
    assert w.tiramisu_hip_rms_norm(None, None, p, p, None, None, None, 4, 8, 0, 0, 1e-6, 2, 2) == 1
    assert w.tiramisu_hip_quantize_rows(p, p, None, 4, 8, 0, 2) == 1
    assert w.tiramisu_hip_rms_norm_backward(p, p, p, None, None, p, p, 4, 8, 0, 0, 0, 2) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 4, 8, far, 0, 0, 0, 0, 2, 2) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 4, 8, 1 << 22, 0, 0, 0, 0, 2, 2) == 1   # rows of 8 MiB
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 4, 8, 8, 0, 0, 0, 9, 2, 2) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 4, 8, 8, 0, 0, 0, 0, 2, 1) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 4, 8, 8, 0, 0, 0, 0, 0, 0) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, p, p, None, 4, 8, 8, 0, 0, 0, 0, 3, 2) == 1
    assert w.tiramisu_hip_linear(p, None, None, None, None, None, p, None, 4, 8, 8, 0, 0, 0, 0, 2, 2) == 1
    assert w.tiramisu_hip_gated_linear(p, p, p, None, None, None, p, p, None, 4, 8, 8, 0, 0, 0, 4, 2, 2) == 1
    assert w.tiramisu_hip_linear_backward(p, p, p, None, p, p, None, 4, 8, 8, 0, 0, 0, 0, 1, 2) == 1
    assert w.tiramisu_hip_linear_backward(p, p, p, None, p, p, None, 4, 8, 8, 0, 0, 0, 0, 0, 3) == 1
    assert w.tiramisu_hip_gated_linear_backward(p, p, p, p, p, p, p, p, None, 4, 8, 8, 0, 0, 0, 0, 0, 0, 4, 2) == 1
    assert w.tiramisu_hip_linear(p, p, None, None, None, None, p, None, 1 << 29, 1 << 9, 8, 0, 0, 0, 0, 2, 2) == 1     # 2^26 tiles
    assert w.tiramisu_hip_rms_norm(p, None, p, p, None, None, None, 4, 1 << 27, 0, 0, 1e-6, 2, 2) == 1
    messages = capfd.readouterr().err.strip().splitlines()
    assert len(messages) == 20 and all(m.startswith("Error at tiramisu_hip_") for m in messages)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(8200, 8195), (8192, 8191), (8192, 8192)])
def test_gradients_of_weights_around_the_size_that_goes_past_the_caches(N, K):
    """2^27 bytes of weights' gradients and some less or more, dense rows at odd elements among them."""
    M, dtype, g = 70, torch.bfloat16, generator(113)
    x, w, dy = normal((M, K), dtype, g), normal((N, K), dtype, g, K ** -0.5), normal((M, N), dtype, g)
    xd, dd = x.double(), dy.double()
    exact = dd.t() @ xd
    close(operators.linear_backward(dy, x, w).dweight, exact, backward_bound(dtype, exact, M, dd.t().abs() @ xd.abs()), "dweight")
    n = N // 2
    gate, up = normal((M, n), dtype, g), normal((M, n), dtype, g)
    got = operators.gated_linear_backward(dy[:, :n].contiguous(), x, w[:n], w[n:], gate, up, activation="none")
    for ours, dz, name in ((got.dgate_weight, dd[:, :n] * up.double(), "dgate_weight"), (got.dup_weight, dd[:, :n] * gate.double(), "dup_weight")):
        exact = dz.t() @ xd
        close(ours, exact, backward_bound(dtype, exact, M, dz.t().abs() @ xd.abs()), name)
