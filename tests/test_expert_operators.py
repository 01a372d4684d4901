"""The operators of a feed-forward sublayer with experts (tiramisu_amd/operators.py: route, the products of grouped rows, combine) against their definitions in 64 bits.

Tolerances are those of test_operators.py, element by element.  A router's weight is exp(z - most) over a sum: the difference is rounded once, which the exponential turns into
|z - most| 2^-24 of itself, the exponential is within two units (2 x 2^-23), the sum of n terms adds n roundings and the quotient one."""
import json
import math

import pytest
import torch

import host_runtime
import test_operators as definitions
from tiramisu_amd import operators, runtime
from test_operators import F8, HALVES, backward_bound, close, exact_activation, exact_slope, generator, normal, rounded, sum_error

WIDE = [torch.float32, torch.float16, torch.bfloat16]


# ---------------------------------------------------------------- route

def exact_route(logits, k, normalise):
    """By counting, one choice after the other: (experts, weights in 64 bits, offsets, rows, places, bound of the weights)"""
    z = logits.double().reshape(-1, logits.shape[-1])
    tokens, count = z.shape
    key = torch.where(z.isnan(), math.inf, z.clamp(-1e300, 1e300))          # NaN above plus infinity, minus infinity below everything
    key = torch.where(z == -math.inf, -math.inf, key)
    number, experts = torch.arange(count, device=z.device), []
    for _ in range(k):
        best = key.max(1, keepdim=True).values
        first = torch.where(key == best, number, count).min(1).values
        experts.append(torch.where(best[:, 0] == -math.inf, -1, first))
        key = key.scatter(1, first[:, None], -math.inf)
    experts = torch.stack(experts, 1)
    there = experts >= 0
    chosen = torch.where(there, z.gather(1, experts.clamp(min=0)), -math.inf)
    of = chosen if normalise else z
    most = torch.where(there[:, :1], chosen[:, :1], 0.0)
    total = torch.where(of == -math.inf, 0.0, torch.exp(of - most)).sum(1, keepdim=True)
    weights = torch.where(there, torch.exp(chosen - most) / total, 0.0)
    bound = torch.where(there, weights * 2.0 ** -24 * ((of - most).abs().nan_to_num(0, 0, 0).amax(1, keepdim=True) + (chosen - most).abs().nan_to_num(0, 0, 0) + of.shape[1] + 16), 0.0) + 2.0 ** -149
    flat = experts.view(-1)
    order = torch.argsort(torch.where(flat < 0, count, flat), stable=True)
    placed = int(there.sum())
    places = torch.full((tokens * k,), -1, device=z.device)
    places[order[:placed]] = torch.arange(placed, device=z.device)
    rows = torch.full((tokens * k,), -1, device=z.device)
    rows[:placed] = order[:placed] // k
    offsets = torch.stack([(flat.view(1, -1) < e).sum() - (flat < 0).sum() for e in range(count + 1)])
    return experts, weights, offsets, rows, places.view(tokens, k), bound


def router_logits(tokens, experts, dtype, seed):
    """With ties, padding (all minus infinity) and masked experts."""
    g = generator(seed)
    z = torch.randn((tokens, experts), device="cuda", generator=g) * 2
    if tokens > 2:
        z[1] = -math.inf
        z[2] = z[2].round()
        z[2, z[2] < 0] = -math.inf
        z[tokens // 2] = 0.5
        z[tokens // 2, ::2] = -0.0
        z[-1] *= 30
    return z.to(dtype)


ROUTES = [(1, 1, 1), (1, 64, 8), (3, 7, 7), (5, 16, 16), (5, 17, 3), (16, 128, 8), (40, 129, 2), (257, 33, 5), (300, 200, 16), (600, 1024, 16), (700, 1000, 4), (5000, 128, 8), (20001, 60, 6), (9000, 300, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("tokens,experts,k", ROUTES)
def test_route(tokens, experts, k, dtype):
    z = router_logits(tokens, experts, dtype, tokens + experts)
    for normalise in (True, False):
        chosen, weights, offsets, rows, places, bound = exact_route(z, k, normalise)
        got = operators.route(z, k, normalise=normalise)
        assert got.experts.dtype == got.offsets.dtype == got.rows.dtype == got.places.dtype == torch.int32
        for name, ours, exact in (("experts", got.experts, chosen), ("offsets", got.offsets, offsets), ("rows", got.rows, rows), ("places", got.places, places)):
            assert ours.shape == exact.shape and torch.equal(ours.long(), exact), name
        close(got.weights, weights, bound, "weights")
        assert all(torch.equal(a, b) for a, b in zip(got, operators.route(z, k, normalise=normalise)))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [8, 1000])
def test_route_of_logits_that_are_not_finite(tokens):
    """NaN is before everything and makes its row's weights NaN, as plus infinity does; the other rows are what they are without."""
    z = router_logits(tokens, 20, torch.float32, 3)
    clean = operators.route(z, 3)
    z[4, 7], z[5, 11], z[5, 3], z[6, 0] = math.nan, math.nan, math.inf, math.inf
    got = operators.route(z, 3)
    assert int(got.experts[4, 0]) == 7 and [int(e) for e in got.experts[5, :2]] == [11, 3] and int(got.experts[6, 0]) == 0
    assert bool(torch.isnan(got.weights[4]).all()) and bool(torch.isnan(got.weights[5]).all()) and bool(torch.isnan(got.weights[6, 0]))
    others = [t for t in range(tokens) if t not in (4, 5, 6)]
    assert torch.equal(got.experts[others], clean.experts[others]) and torch.equal(got.weights[others], clean.weights[others])


@pytest.mark.gpu
def test_route_of_no_tokens_and_of_leading_dimensions():
    none = operators.route(torch.empty((0, 9), device="cuda"), 2)
    assert not bool(none.offsets.any()) and none.offsets.shape == (10,) and none.rows.shape == (0,) and none.places.shape == (0, 2)
    wide = torch.randn((4, 70, 40), device="cuda", generator=generator(5)).bfloat16()
    z = wide[..., 3:36]
    got, packed = operators.route(z, 4), operators.route(z.reshape(280, 33), 4)
    assert got.experts.shape == (4, 70, 4) and got.places.shape == (4, 70, 4)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, packed))
    d = torch.randn((4, 70, 4), device="cuda", generator=generator(6))
    assert torch.equal(operators.route_backward(d, z, got.experts).view(280, 33), operators.route_backward(d.view(280, 4), z.reshape(280, 33), packed.experts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("tokens,experts,k", ROUTES)
def test_route_backward(tokens, experts, k, dtype):
    z = router_logits(tokens, experts, dtype, 7 + tokens)
    g = torch.randn((tokens, k), device="cuda", generator=generator(11))
    for normalise in (True, False):
        chosen, w, _, _, _, bound = exact_route(z, k, normalise)
        there = chosen >= 0
        gd = torch.where(there, g.double(), 0.0)
        dot, size = (w * gd).sum(1, keepdim=True), (w * gd.abs()).sum(1, keepdim=True)
        relative = 2.0 ** -24 * ((bound / 2.0 ** -24 / w.clamp(min=1e-300)).clamp(max=1e6).masked_fill(~there, 0).amax(1, keepdim=True) + k + 8)
        exact = torch.zeros((tokens, experts + 1), dtype=torch.float64, device="cuda")
        error = exact.clone()
        index = torch.where(there, chosen, experts)
        if normalise:
            exact.scatter_(1, index, w * (gd - dot))
            error.scatter_(1, index, w * (gd.abs() + size) * 3 * relative)
        else:
            p = torch.where(there[:, :1] & (z != -math.inf), torch.exp(z.double() - torch.where(there[:, :1], z.double().amax(1, keepdim=True), 0.0)), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            exact[:, :-1] = -p * dot
            error[:, :-1] = p * size * 3 * (relative + 2.0 ** -24 * (z.double() - z.double().amax(1, keepdim=True)).abs().nan_to_num(0, 0, 0))
            exact.scatter_add_(1, index, w * gd)
            error.scatter_add_(1, index, w * gd.abs() * 3 * relative)
        exact, error = exact[:, :-1], error[:, :-1]
        # (numbers below 2^-126 have fewer bits)
        close(operators.route_backward(g, z, chosen.int(), normalise=normalise), exact, rounded(exact, error + 2.0 ** -140, dtype), "dlogits")


@pytest.mark.gpu
def test_route_backward_against_differences():
    z = torch.randn((5, 12), device="cuda", generator=generator(13))
    g, d = torch.randn((5, 4), device="cuda", generator=generator(14)), torch.randn((5, 12), device="cuda", generator=generator(15), dtype=torch.float64)
    for normalise in (True, False):
        experts = operators.route(z, 4, normalise=normalise).experts

        def value(z):
            p = torch.softmax(z, 1).gather(1, experts.long())
            return float(((p / p.sum(1, keepdim=True) if normalise else p) * g.double()).sum())

        grad = operators.route_backward(g, z, experts, normalise=normalise)
        h = 1e-5
        difference = (value(z.double() + h * d) - value(z.double() - h * d)) / (2 * h)
        # truncation h^2 of a third derivative of order 1 an element, rounding 2^-50 / h, and the gradients' own 32 bits
        bound = 60 * (h * h * 50 + 2.0 ** -50 / h) + float((d.abs() * grad.double().abs()).sum() + 60) * 40 * 2.0 ** -24
        assert abs(difference - float((grad.double() * d).sum())) <= bound


# ---------------------------------------------------------------- products of grouped rows

# places of each group, behind the last group's, N, K.  Empty groups, single rows, tiles that end inside a group, one group, many.
GROUPS = [([1], 0, 1, 1), ([0, 5, 0, 1, 17], 3, 17, 33), ([0, 0], 4, 40, 64), ([3, 2, 0, 16, 33], 0, 40, 8), ([70], 0, 100, 72), ([300, 0, 1, 129, 64], 30, 130, 200), ([0, 0, 257], 1, 300, 129),
          ([1] * 70 + [0] * 30 + [2] * 40, 5, 24, 1001), ([40, 7, 90], 100, 520, 300), ([600, 520, 0, 700], 0, 264, 136), ([2, 1, 0, 1], 0, 300, 2050), ([500] * 3 + [3], 2, 66, 71)]


def grouped_inputs(sizes, behind, N, K, dtype, seed, weights=1, picked=False):
    """offsets, rows (None), x, its scale, weights, their scales, and in 64 bits: the places' rows and the weights."""
    g = generator(seed)
    S, E = sum(sizes) + behind, len(sizes)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(E + 1)], device="cuda", dtype=torch.int32)
    rows, T = None, S
    if picked:
        T = S // 2 + 3
        rows = torch.randint(0, T, (S,), device="cuda", generator=g, dtype=torch.int32)
        rows[::7] = -1
        rows[3::11] = T
    x, ws = torch.randn((T, K), device="cuda", generator=g), [torch.randn((E, N, K), device="cuda", generator=g) * max(1, K) ** -0.5 for _ in range(weights)]
    if dtype == F8:
        x, xs = definitions.in_8_bits(x)
        pairs = [definitions.in_8_bits(w.view(E * N, K)) for w in ws]
        ws, scales = [q.view(E, N, K) for q, _ in pairs], [s.view(E, N) for _, s in pairs]
        xd, wd = x.double() * xs.double()[:, None], [w.double() * s.double()[..., None] for w, s in zip(ws, scales)]
    else:
        x, xs, ws, scales = x.to(dtype), None, [w.to(dtype) for w in ws], [None] * weights
        xd, wd = x.double(), [w.double() for w in ws]
    if picked:
        there = (rows >= 0) & (rows < T)
        xd = torch.where(there[:, None], xd[rows.clamp(0, T - 1).long()], 0.0)
    return offsets, rows, x, xs, ws, scales, xd, wd


def by_group(sizes, behind, xd, wd, of):
    """of(rows, weight) group by group; zeros behind"""
    out, at = [], 0
    for e, n in enumerate(sizes):
        out.append(of(xd[at:at + n], wd[e]))
        at += n
    return torch.cat(out + [torch.zeros((behind, out[0].shape[1]), dtype=torch.float64, device="cuda")])


def product(x, w):
    return x @ w.t()


def sizes_of(x, w):
    return x.abs() @ w.abs().t()


def cut(dtype):
    return lambda x, w: definitions.cut_off(x, w, dtype) if dtype == F8 and len(x) and x.shape[1] else torch.zeros((len(x), len(w)), dtype=torch.float64, device="cuda")


def check_grouped(sizes, behind, N, K, dtype, out=None):
    out = out or (torch.float16 if dtype == torch.float16 else torch.bfloat16)
    for picked in (False, True):
        offsets, rows, x, xs, ws, scales, xd, wds = grouped_inputs(sizes, behind, N, K, dtype, N + K, weights=2, picked=picked)
        z = [by_group(sizes, behind, xd, wd, product) for wd in wds]
        error = [sum_error(K, by_group(sizes, behind, xd, wd, sizes_of)) + by_group(sizes, behind, xd, wd, cut(dtype)) for wd in wds]
        y = operators.grouped_linear(x, ws[0], offsets, rows=rows, x_scale=xs, weight_scale=scales[0], dtype=out)
        assert y.dtype == out
        close(y, z[0], rounded(z[0], error[0], out), "y")
        for i, activation in enumerate(("silu", "gelu")):
            got = operators.grouped_gated_linear(x, ws[0], ws[1], offsets, rows=rows, activation=activation, x_scale=xs, gate_scale=scales[0], up_scale=scales[1], dtype=out, keep_pre=i == 0)
            a = exact_activation(activation, z[0])
            h = a * z[1]
            ea = 1.13 * error[0] + 2.0 ** -22 * (z[0].abs() + 1)
            close(got.h, h, rounded(h, ea * (z[1].abs() + error[1]) + a.abs() * error[1] + 2.0 ** -23 * h.abs(), out), "%s h" % activation)
            if i == 0:
                close(got.gate, z[0], rounded(z[0], error[0], out), "gate")
                close(got.up, z[1], rounded(z[1], error[1], out), "up")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("sizes,behind,N,K", GROUPS)
def test_grouped(sizes, behind, N, K, dtype):
    check_grouped(sizes, behind, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,behind,N,K", GROUPS[1:6])
def test_grouped_8_bits_in_float16(sizes, behind, N, K):
    check_grouped(sizes, behind, N, K, F8, torch.float16)


def check_grouped_backward(sizes, behind, N, K, dtype):
    for picked in (False, True):
        offsets, rows, x, _, (wg, wu), _, xd, (gd, ud) = grouped_inputs(sizes, behind, N, K, dtype, 31 + N, weights=2, picked=picked)
        g = generator(37)
        S = sum(sizes) + behind
        dy, gate, up = normal((S, N), dtype, g), normal((S, N), dtype, g, 2.0), normal((S, N), dtype, g)
        if behind:
            # (nothing behind the groups counts)
            dy[-behind:], gate[-behind:], up[-behind:] = math.nan, math.inf, math.nan
        at = [sum(sizes[:e]) for e in range(len(sizes))]
        spans = [slice(a, a + n) for a, n in zip(at, sizes)]

        def of_weights(dz, xd):
            return torch.stack([dz[s].t() @ xd[s] for s in spans])

        def of_rows(dz, wd):
            return by_group(sizes, behind, dz, wd, lambda d, w: d @ w)

        most = max(sizes) if sizes else 0
        got = operators.grouped_linear_backward(dy, x, wg, offsets, rows=rows)
        d = dy.double()
        exact = of_rows(d, gd)
        close(got.dx, exact, backward_bound(dtype, exact, N, of_rows(d.abs(), gd.abs())) + torch.zeros_like(exact), "dx")
        exact = of_weights(d, xd)
        close(got.dweight, exact, backward_bound(dtype, exact, most, of_weights(d.abs(), xd.abs())), "dweight")
        for activation in ("silu", "relu"):
            got = operators.grouped_gated_linear_backward(dy, x, wg, wu, gate, up, offsets, rows=rows, activation=activation)
            zd = gate.double()
            slope = (zd > 0).double() if activation == "relu" else exact_slope(activation, zd)
            dgate, dup = d * up.double() * slope, d * exact_activation(activation, zd)
            slack = 16 * 2.0 ** -24 * d.abs() * (1 + up.double().abs() + zd.abs()) / definitions.ROUNDOFF[dtype]
            sg, su = dgate.abs() + slack, dup.abs() + slack
            exact = of_rows(dgate, gd) + of_rows(dup, ud)
            close(got.dx, exact, backward_bound(dtype, exact, 2 * N, of_rows(sg, gd.abs()) + of_rows(su, ud.abs())), "%s dx" % activation)
            for ours, dz, s, name in ((got.dgate_weight, dgate, sg, "dgate_weight"), (got.dup_weight, dup, su, "dup_weight")):
                exact = of_weights(dz, xd)
                close(ours, exact, backward_bound(dtype, exact, most, of_weights(s, xd.abs())), "%s %s" % (activation, name))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("sizes,behind,N,K", GROUPS)
def test_grouped_backward(sizes, behind, N, K, dtype):
    check_grouped_backward(sizes, behind, N, K, dtype)


@pytest.mark.gpu
def test_grouped_of_no_rows():
    w = normal((3, 40, 64), torch.bfloat16, generator(3))
    x, offsets = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16), torch.zeros(4, device="cuda", dtype=torch.int32)
    e = torch.empty((0, 40), device="cuda", dtype=torch.bfloat16)
    assert operators.grouped_linear(x, w, offsets).shape == (0, 40) and operators.grouped_gated_linear(x, w, w, offsets).h.shape == (0, 40)
    got = operators.grouped_linear_backward(e, x, w, offsets)
    assert got.dx.shape == (0, 64) and got.dweight.shape == w.shape and not bool(got.dweight.any())
    got = operators.grouped_gated_linear_backward(e, x, w, w, e, e, offsets)
    assert not bool(got.dgate_weight.any()) and not bool(got.dup_weight.any())
    # places, but no token that they could take, and no terms
    rows = torch.zeros(70, device="cuda", dtype=torch.int32)
    ends = torch.tensor([0, 20, 20, 60], device="cuda", dtype=torch.int32)
    for n in (70, 9):
        assert not bool(operators.grouped_linear(x, w, ends.clamp(max=n), rows=rows[:n]).any())
    assert not bool(operators.grouped_linear(torch.empty((70, 0), device="cuda", dtype=torch.bfloat16), w[..., :0], ends).any())
    dy = normal((70, 40), torch.bfloat16, generator(4))
    assert not bool(operators.grouped_linear_backward(dy, x, w, ends, rows=rows).dweight.any())


@pytest.mark.gpu
@pytest.mark.parametrize("S", [9, 300])
def test_offsets_that_lead_nowhere(S):
    """Whatever the offsets hold, nothing outside of the operands is read or written: groups are cut off at the rows that there are."""
    g = generator(5)
    x, w, dy = normal((S, 70), torch.bfloat16, g), normal((3, 40, 70), torch.bfloat16, g), normal((S, 40), torch.bfloat16, g)
    for ends in ([-5, 4, 6, 1 << 30], [0, 8, 2, S], [S, 0, 0, 0], [-2 ** 31, 2 ** 31 - 1, -1, 7]):
        offsets = torch.tensor(ends, device="cuda", dtype=torch.int32)
        assert operators.grouped_linear(x, w, offsets).shape == (S, 40)
        assert operators.grouped_linear_backward(dy, x, w, offsets).dweight.shape == w.shape
    cut_off = operators.grouped_linear(x, w, torch.tensor([-5, 4, 6, 1 << 30], device="cuda", dtype=torch.int32))
    assert torch.equal(cut_off, operators.grouped_linear(x, w, torch.tensor([0, 4, 6, S], device="cuda", dtype=torch.int32)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("sizes,N,K,first", [([2, 0, 3], 33, 70, 0), ([40, 30], 66, 71, 1), ([130, 0, 60, 4], 140, 200, 3)])
def test_grouped_operands_within_larger_tensors(sizes, N, K, first, dtype):
    """Rows that go on into infinities and NaN, that begin at odd elements and are odd strides apart: results are those of dense operands."""

    def within(t, low, high):
        big = torch.full((t.shape[0] + 2, *t.shape[1:-1], t.shape[-1] + low + high), math.nan, device="cuda").to(t.dtype)
        big[1:-1, ..., low:low + t.shape[-1]] = t
        return big[1:-1, ..., low:low + t.shape[-1]]

    for picked in (False, True):
        offsets, rows, x, xs, ws, scales, _, _ = grouped_inputs(sizes, 3, N, K, dtype, 47, weights=2, picked=picked)
        xv, wv = within(x, first, 5), [within(w, first, 2) for w in ws]
        a = operators.grouped_linear(x, ws[0], offsets, rows=rows, x_scale=xs, weight_scale=scales[0])
        assert torch.equal(a, operators.grouped_linear(xv, wv[0], offsets, rows=rows, x_scale=xs, weight_scale=scales[0]))
        a = operators.grouped_gated_linear(x, ws[0], ws[1], offsets, rows=rows, x_scale=xs, gate_scale=scales[0], up_scale=scales[1])
        assert torch.equal(a.h, operators.grouped_gated_linear(xv, wv[0], wv[1], offsets, rows=rows, x_scale=xs, gate_scale=scales[0], up_scale=scales[1]).h)
        if dtype == F8:
            continue
        g = generator(48)
        S = sum(sizes) + 3
        dy, gate, up = [normal((S, N), dtype, g) for _ in range(3)]
        a, b = operators.grouped_linear_backward(dy, x, ws[0], offsets, rows=rows), operators.grouped_linear_backward(within(dy, first, 2), xv, wv[0], offsets, rows=rows)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        a = operators.grouped_gated_linear_backward(dy, x, ws[0], ws[1], gate, up, offsets, rows=rows)
        b = operators.grouped_gated_linear_backward(within(dy, first, 2), xv, wv[0], wv[1], within(gate, first, 2), within(up, first, 2), offsets, rows=rows)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_infinities_stay_in_their_rows_and_groups():
    for sizes in ([3, 2, 4], [130, 20, 150]):
        offsets, _, x, _, (w, v), _, _, _ = grouped_inputs(sizes, 0, 40, 100, torch.bfloat16, 53, weights=2)
        clean, clean_h = operators.grouped_linear(x, w, offsets), operators.grouped_gated_linear(x, w, v, offsets).h
        a = sizes[0]
        x[a, 99], w[2, 5, 0] = math.inf, math.nan
        for got, was in ((operators.grouped_linear(x, w, offsets), clean), (operators.grouped_gated_linear(x, w, v, offsets).h, clean_h)):
            assert not bool(torch.isfinite(got[a]).any()) and bool(torch.isnan(got[a + sizes[1]:, 5]).all())
            was = was.clone()
            was[a], was[a + sizes[1]:, 5] = 0, 0
            got[a], got[a + sizes[1]:, 5] = 0, 0
            assert torch.equal(got, was)


@pytest.mark.gpu
def test_picked_rows_beyond_2_gib():
    """Rows a long way apart, so that the last begin behind 2^32 bytes: such rows are gathered ahead of the tiles, and read in place by the kernel of few rows."""
    T, N, K, step = 2400, 72, 80, 1 << 20
    g = generator(67)
    far = torch.empty(T * step, dtype=torch.bfloat16, device="cuda").view(T, step)[:, :K]
    x = normal((T, K), torch.bfloat16, g)
    far.copy_(x)
    w = normal((4, N, K), torch.bfloat16, g, 0.1)
    for S in (16, 500):
        rows = torch.randint(T - 600, T, (S,), device="cuda", generator=g, dtype=torch.int32)
        offsets = torch.tensor([0, S // 3, S // 2, S // 2, S], device="cuda", dtype=torch.int32)
        assert torch.equal(operators.grouped_linear(far, w, offsets, rows=rows), operators.grouped_linear(x, w, offsets, rows=rows))
        dy = normal((S, N), torch.bfloat16, g)
        assert torch.equal(operators.grouped_linear_backward(dy, far, w, offsets, rows=rows).dweight, operators.grouped_linear_backward(dy, x, w, offsets, rows=rows).dweight)


@pytest.mark.gpu
@pytest.mark.parametrize("each", [1, 9])
def test_as_many_groups_as_there_may_be(each):
    check_grouped([each * (i % 3) for i in range(1024)], 5, 40, 72, torch.bfloat16)
    check_grouped_backward([each * (i % 3) for i in range(1024)], 5, 40, 72, torch.bfloat16)


def linear_bound(z, x, w):
    return rounded(z, sum_error(x.shape[1], x.abs() @ w.abs().t()), torch.bfloat16)


@pytest.mark.gpu
def test_weights_beyond_4_gib():
    """The last of 40 groups' weights begin behind 2^32 bytes, and so does its gradient."""
    E, N = 40, 8192
    g = generator(73)
    w = torch.empty((E, N, N), dtype=torch.bfloat16, device="cuda")
    w[-1] = normal((N, N), torch.bfloat16, g, N ** -0.5)
    wd = w[-1].double()
    for S, n in ((30, 20), (400, 130)):                   # few rows, and tiles
        x, dy = normal((S, N), torch.bfloat16, g), normal((S, N), torch.bfloat16, g)
        offsets = torch.full((E + 1,), S - n, dtype=torch.int32, device="cuda")
        offsets[-1] = S
        offsets[0] = 0
        w[0] = 0
        xd, dd = x[-n:].double(), dy[-n:].double()
        z = xd @ wd.t()
        y = operators.grouped_linear(x, w, offsets)
        close(y[-n:], z, linear_bound(z, xd, wd), "y")
        assert not bool(y[:-n].any())
        got = operators.grouped_linear_backward(dy, x, w, offsets)
        z = dd @ wd
        close(got.dx[-n:], z, linear_bound(z, dd, wd.t()), "dx")
        z = dd.t() @ xd
        close(got.dweight[-1], z, linear_bound(z, dd.t(), xd.t()), "dweight")
        assert not bool(got.dweight[1:-1].any())


@pytest.mark.gpu
def test_results_beyond_4_gib():
    """Places whose rows begin behind 2^32 bytes of what is stored, kept, read again and combined."""
    S, N, K, last = 600000, 4096, 24, 300
    g = generator(79)
    x, w, v = normal((S, K), torch.bfloat16, g), normal((2, N, K), torch.bfloat16, g), normal((2, N, K), torch.bfloat16, g)
    offsets = torch.tensor([0, S - last, S], dtype=torch.int32, device="cuda")
    xd, wd, vd = x[-last:].double(), w[1].double(), v[1].double()
    z, u = xd @ wd.t(), xd @ vd.t()
    y = operators.grouped_linear(x, w, offsets)
    close(y[-last:], z, linear_bound(z, xd, wd), "y")
    got = operators.grouped_gated_linear(x, w, v, offsets, keep_pre=True)
    close(got.gate[-last:], z, linear_bound(z, xd, wd), "gate")
    close(got.up[-last:], u, linear_bound(u, xd, vd), "up")
    back = operators.grouped_linear_backward(y, x, w, offsets)
    yd = y[-last:].double()
    z = yd @ wd
    close(back.dx[-last:], z, linear_bound(z, yd, wd.t()), "dx")
    z = yd.t() @ xd
    close(back.dweight[1], z, linear_bound(z, yd.t(), xd.t()), "dweight")
    places = torch.arange(S - 8, S, dtype=torch.int32, device="cuda").view(4, 2)
    weights = torch.randn((4, 2), device="cuda", generator=g)
    sums = (y[-8:].double().view(4, 2, N) * weights.double()[..., None]).sum(1)
    close(operators.combine(y, places, weights), sums, rounded(sums, 4 * 2.0 ** -24 * (y[-8:].double().view(4, 2, N) * weights.double()[..., None]).abs().sum(1), torch.bfloat16), "combined")
    owners = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    owners[-8:] = torch.arange(4, device="cuda", dtype=torch.int32).repeat_interleave(2)
    dy = normal((4, N), torch.bfloat16, g)
    c = operators.combine_backward(dy, y, places, weights, owners)
    z = (dy.double()[:, None] * weights.double()[..., None]).view(8, N)
    close(c.dx[-8:], z, rounded(z, 2.0 ** -24 * z.abs(), torch.bfloat16), "combine's dx")
    assert not bool(c.dx[:-8].any())


@pytest.mark.gpu
def test_terms_of_a_group_shared_by_workgroups_and_picked():
    """The weights' gradient alone, whose workgroups each have more terms than an index in LDS holds at a time."""
    S, T, N, K = 300000, 5000, 72, 80
    g = generator(83)
    dy, x = normal((S, N), torch.bfloat16, g), normal((T, K), torch.bfloat16, g)
    rows = torch.randint(-1, T + 1, (S,), device="cuda", generator=g, dtype=torch.int32)
    offsets = torch.tensor([0, S - 70, S - 9], dtype=torch.int32, device="cuda")
    dweight = torch.full((2, N, K), math.nan, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    assert runtime.wrappers().tiramisu_hip_grouped_linear_backward(dy.data_ptr(), x.data_ptr(), None, offsets.data_ptr(), rows.data_ptr(), None, dweight.data_ptr(), S, T, 2, N, K, 0, 0, 0, 2) == 0
    torch.cuda.synchronize()
    there = (rows >= 0) & (rows < T)
    xd, dd = torch.where(there[:, None], x.double()[rows.clamp(0, T - 1).long()], 0.0), dy.double()
    for e, (first, end) in enumerate(((0, S - 70), (S - 70, S - 9))):
        a, b = dd[first:end].t(), xd[first:end].t()
        z = a @ b.t()
        close(dweight[e], z, linear_bound(z, a, b), "dweight")


# ---------------------------------------------------------------- combine

COMBINES = [(1, 1, 1, 1), (3, 2, 7, 5), (5, 8, 64, 100), (40, 3, 1430, 130), (130, 9, 1001, 2000), (17, 20, 264, 340), (9, 4, 4100, 36), (2, 0, 40, 3)]


def combine_inputs(tokens, k, N, places, dtype, seed):
    """Places in any order, some of them none of x's; the token of each."""
    g = generator(seed)
    at = torch.full((tokens * k,), -1, device="cuda", dtype=torch.int32)
    used = torch.randperm(places, device="cuda", generator=g)[:tokens * k].int()
    at[torch.randperm(tokens * k, device="cuda", generator=g)[:len(used)]] = used
    at[::5] = -1
    if tokens * k > 3:
        at[3] = places
    rows = torch.full((places,), -1, device="cuda", dtype=torch.int32)
    there = (at >= 0) & (at < places)
    rows[at[there].long()] = (torch.nonzero(there)[:, 0] // max(1, k)).int()
    return at.view(tokens, k), rows, normal((places, N), dtype, g), torch.randn((tokens, k), device="cuda", generator=g), normal((tokens, N), dtype, g), normal((tokens, N), dtype, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("tokens,k,N,places", COMBINES)
def test_combine(tokens, k, N, places, dtype):
    at, rows, x, w, r, _ = combine_inputs(tokens, k, N, places, dtype, 3 + N)
    if len(x) > 2 and k:
        x[int(torch.nonzero(rows < 0)[0])] = math.nan if bool((rows < 0).any()) else 0      # (a row that is nobody's)
    there = (at >= 0) & (at < places)
    gathered = torch.where(there[..., None], x.double()[at.clamp(0, places - 1).long()], 0.0)
    for weights in (w, None):
        for residual in (r, None):
            terms = gathered if weights is None else gathered * w.double()[..., None]
            y, size = terms.sum(1), terms.abs().sum(1)
            if residual is not None:
                y, size = y + r.double(), size + r.double().abs()
            got = operators.combine(x, at, weights=weights, residual=residual)
            close(got, y, rounded(y, (k + 2) * 2.0 ** -24 * size, dtype), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("tokens,k,N,places", COMBINES)
def test_combine_backward(tokens, k, N, places, dtype):
    at, rows, x, w, dy, _ = combine_inputs(tokens, k, N, places, dtype, 5 + N)
    there = (at >= 0) & (at < places)
    for weights in (w, None):
        got = operators.combine_backward(dy, x, at, weights, rows)
        dx = torch.zeros((places, N), dtype=torch.float64, device="cuda")
        factor = torch.ones_like(w) if weights is None else w
        dx[at[there].long()] = (factor.double()[..., None] * dy.double()[:, None])[there]
        close(got.dx, dx, rounded(dx, 2.0 ** -24 * dx.abs(), dtype), "dx")
        assert (got.dweights is None) == (weights is None)
        if weights is not None:
            terms = torch.where(there[..., None], x.double()[at.clamp(0, places - 1).long()], 0.0) * dy.double()[:, None]
            close(got.dweights, terms.sum(2), (N + 4) * 2.0 ** -24 * terms.abs().sum(2) + 2.0 ** -140, "dweights")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [40, 1001])
def test_choices_left_out_after_the_route(N):
    """A choice that is dropped by -1 in `places`, with `rows` as they were: its row has a gradient of zeros."""
    g = generator(89)
    r = operators.route(torch.randn((150, 7), device="cuda", generator=g), 3)
    places = r.places.masked_fill(torch.rand((150, 3), device="cuda", generator=g) < 0.3, -1)
    x, dy = normal((450, N), torch.bfloat16, g), normal((150, N), torch.bfloat16, g)
    dropped = torch.full((450,), True, device="cuda")
    dropped[places[places >= 0].long()] = False
    for _ in range(3):
        torch.full((450, N), math.nan, device="cuda", dtype=torch.bfloat16)          # (what the allocator hands out next)
        got = operators.combine_backward(dy, x, places, r.weights, r.rows)
        assert not bool(got.dx[dropped].any()) and bool(torch.isfinite(got.dx.float()).all())
        assert bool((got.dweights[places < 0] == 0).all())


@pytest.mark.gpu
def test_combine_of_strided_rows_and_leading_dimensions():
    at, rows, x, w, r, dy = combine_inputs(12, 3, 301, 30, torch.bfloat16, 9)
    wide = torch.full((30, 400), math.nan, device="cuda", dtype=torch.bfloat16)
    wide[:, 7:308] = x
    wide_r = torch.full((3, 4, 340), math.nan, device="cuda", dtype=torch.bfloat16)
    wide_r[..., 5:306] = r.view(3, 4, 301)
    y = operators.combine(wide[:, 7:308], at.view(3, 4, 3), weights=w.view(3, 4, 3), residual=wide_r[..., 5:306])
    assert y.shape == (3, 4, 301) and torch.equal(y.view(12, 301), operators.combine(x, at, weights=w, residual=r))
    wide_r[..., 5:306] = dy.view(3, 4, 301)
    a, b = operators.combine_backward(wide_r[..., 5:306], wide[:, 7:308], at.view(3, 4, 3), w.view(3, 4, 3), rows), operators.combine_backward(dy, x, at, w, rows)
    assert torch.equal(a.dx, b.dx) and torch.equal(a.dweights.view(12, 3), b.dweights)


@pytest.mark.gpu
def test_combine_of_no_tokens_or_rows():
    none = torch.empty((0, 4), device="cuda", dtype=torch.int32)
    x = normal((5, 40), torch.bfloat16, generator(1))
    assert operators.combine(x, none).shape == (0, 40)
    got = operators.combine_backward(x[:0], x, none, torch.empty((0, 4), device="cuda"), torch.full((5,), -1, device="cuda", dtype=torch.int32))
    assert not bool(got.dx.any()) and got.dweights.shape == (0, 4)
    at = torch.zeros((3, 4), device="cuda", dtype=torch.int32)
    assert not bool(operators.combine(x[:0], at).any()) and torch.equal(operators.combine(x[:0], at, residual=x[:3]), x[:3])
    got = operators.combine_backward(x[:3], x[:0], at, torch.ones((3, 4), device="cuda"), torch.empty((0,), device="cuda", dtype=torch.int32))
    assert got.dx.shape == (0, 40) and not bool(got.dweights.any())


# ---------------------------------------------------------------- together

def sublayer(x, router, gate, up, down, k, dy):
    logits = operators.linear(x, router).y
    r = operators.route(logits, k)
    g = operators.grouped_gated_linear(x, gate, up, r.offsets, rows=r.rows, keep_pre=True)
    out = operators.grouped_linear(g.h, down, r.offsets)
    y = operators.combine(out, r.places, weights=r.weights, residual=x)
    c = operators.combine_backward(dy, out, r.places, r.weights, r.rows)
    d = operators.grouped_linear_backward(c.dx, g.h, down, r.offsets)
    e = operators.grouped_gated_linear_backward(d.dx, x, gate, up, g.gate, g.up, r.offsets, rows=r.rows)
    dlogits = operators.route_backward(c.dweights, logits, r.experts)
    back = operators.linear_backward(dlogits, x, router)
    dx = operators.combine(e.dx, r.places, residual=back.dx)
    return y, dx, back.dweight, e.dgate_weight, e.dup_weight, d.dweight


def sublayer_inputs(T, E, hidden, inner, dtype, seed):
    g = generator(seed)
    return [normal((T, hidden), dtype, g), normal((E, hidden), dtype, g, hidden ** -0.5), normal((E, inner, hidden), dtype, g, hidden ** -0.5), normal((E, inner, hidden), dtype, g, hidden ** -0.5),
            normal((E, hidden, inner), dtype, g, inner ** -0.5)], normal((T, hidden), dtype, g)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (30, 6, 3), (700, 5, 2)])
def test_the_sublayer_against_differences(T, E, k):
    """The whole sublayer's gradients along random directions, against central differences of its 64-bit value with the router's choice held."""
    args, dy = sublayer_inputs(T, E, 72, 40, torch.float16, 3)
    experts = operators.route(operators.linear(args[0], args[1]).y, k).experts.long()
    _, *grads = sublayer(*args, k, dy)

    def value(x, router, gate, up, down):
        w = torch.softmax((x @ router.t()).gather(1, experts), 1)
        y = x.clone()
        for e in range(E):
            out = (exact_activation("silu", x @ gate[e].t()) * (x @ up[e].t())) @ down[e].t()
            y = y + (w * (experts == e)).sum(1, keepdim=True) * out
        return float((y * dy.double()).sum())

    at = [t.double() for t in args]
    # (dx is that of the branch; the residual's own is dy)
    grads[0] = grads[0].double() + dy.double()
    for i, grad in enumerate(grads):
        d = torch.randn(grad.shape, device="cuda", generator=generator(5 + i), dtype=torch.float64)
        ends = [value(*[t + (s * 1e-6 * d if j == i else 0) for j, t in enumerate(at)]) for s in (1, -1)]
        difference, ours = (ends[0] - ends[1]) / 2e-6, float((grad.double() * d).sum())
        # some twenty stored intermediates, each off by at most 2^-11 of itself; a gradient is a sum whose terms are larger than it by the square root of their number,
        # which the sum of magnitudes over all elements covers where they are independent
        bound = 24 * 2.0 ** -11 * float((grad.double().abs() * d.abs()).sum())
        print("difference %.6g, gradient %.6g, bound %.3g" % (difference, ours, bound), flush=True)
        assert abs(difference - ours) <= bound, i


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 300])
def test_the_sublayer_in_a_graph(T):
    """Recorded once and replayed on new inputs, which route otherwise, with eager work between the replays."""
    args, dy = sublayer_inputs(T, 12, 136, 72, torch.bfloat16, 7)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        sublayer(*args, 3, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = sublayer(*args, 3, dy)
    for seed in range(4):
        args[0].copy_(normal((T, 136), torch.bfloat16, generator(seed)))
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        for u, v in zip(got, sublayer(*args, 3, dy)):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_two_graphs_beside_each_other():
    """Recorded one after the other on the stream that torch records on, replayed at the same time on two streams: each has scratch of its own."""
    cases = [sublayer_inputs(T, 9, 131, 77, torch.bfloat16, T) for T in (400, 900)]
    expected = [sublayer(*args, 2, dy) for args, dy in cases]
    graphs, results = [], []
    for args, dy in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(sublayer(*args, 2, dy))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for _ in range(10):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for got, was in zip(results, expected):
            assert all(torch.equal(u, v) for u, v in zip(got, was))


@pytest.mark.gpu
def test_calls_follow_the_work_on_a_side_stream():
    args, dy = sublayer_inputs(200, 6, 264, 136, torch.bfloat16, 71)
    x0 = args[0].clone()
    expected = sublayer(x0 * 2, *args[1:], 2, dy)
    torch.cuda.synchronize()
    a = torch.randn((6000, 6000), device="cuda")
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(3):
            a = a @ a * 1e-4                       # keeps the stream busy for some ms
        x = x0 * 2
        got = [t.clone() for t in sublayer(x, *args[1:], 2, dy)]
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, expected))


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Eager calls with scratch (moved operands, shared terms), one stream beside the other: the results of calls on their own."""
    cases = []
    for seed, (S, E, N, K) in enumerate(((9000, 3, 102, 103), (4001, 2, 77, 131))):
        g = generator(91 + seed)
        x, w, dy = normal((S, K), torch.float16, g), normal((E, N, K), torch.float16, g, 0.1), normal((S, N), torch.float16, g)
        offsets = torch.linspace(0, S, E + 1, device="cuda").int()
        cases.append((dy, x, w, offsets))
    expected = [[t.clone() for t in operators.grouped_linear_backward(*c)] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(operators.grouped_linear_backward(*cases[i]))
    torch.cuda.synchronize()
    for results, was in zip(got, expected):
        for r in results:
            assert all(torch.equal(u, v) for u, v in zip(r, was))


@pytest.mark.gpu
def test_shared_terms_in_a_graph():
    g = generator(97)
    x, w, dy = normal((14000, 103), torch.float16, g), normal((3, 192, 103), torch.float16, g, 0.1), normal((14000, 192), torch.float16, g)
    offsets = torch.tensor([0, 5000, 9000, 14000], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out = operators.grouped_linear_backward(dy, x, w, offsets)
    for ends in ([0, 14000, 14000, 14000], [0, 10, 20, 30], [0, 4000, 9001, 13000]):
        offsets.copy_(torch.tensor(ends, dtype=torch.int32))
        dy.copy_(normal(dy.shape, torch.float16, generator(ends[1])))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, operators.grouped_linear_backward(dy, x, w, offsets)))


@pytest.mark.gpu
def test_calls_in_inference_mode():
    args, dy = sublayer_inputs(40, 6, 136, 72, torch.bfloat16, 13)
    expected = sublayer(*args, 2, dy)
    with torch.inference_mode():
        got = sublayer(*args, 2, dy)
        r = operators.route(operators.linear(args[0], args[1]).y, 2)
        assert r.weights.sum(-1).shape == (40,) and int(r.offsets[-1]) == 80
    assert all(torch.equal(u, v) for u, v in zip(got, expected))
    # the results of a route are tensors like others: changed in place, kept by autograd
    r = operators.route(operators.linear(args[0], args[1]).y, 2)
    kept = r.weights.clone()
    scale = torch.ones(2, device="cuda", requires_grad=True)
    (r.weights * scale).sum().backward()
    assert torch.allclose(scale.grad, kept.sum(0), rtol=1e-5)
    r.weights.mul_(2)
    assert torch.equal(r.weights, kept * 2)


@pytest.mark.gpu
def test_launches_are_recorded_by_the_profile():
    args, dy = sublayer_inputs(4, 3, 64, 64, torch.bfloat16, 5)
    records = runtime.profile(lambda: sublayer(*args, 2, dy))
    names = [name[len("tiramisu_hip_"):] for name, _ in records]
    assert names == ["linear", "route", "grouped_gated_linear", "grouped_linear", "combine_rows", "combine_rows_backward", "grouped_linear_backward", "grouped_gated_linear_backward", "route_backward",
                     "linear_backward", "combine_rows"]


# ---------------------------------------------------------------- refusals

def test_what_is_refused_without_a_gpu():
    x, w, o = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((2, 8, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: operators.route(x, 2), lambda: operators.grouped_linear(x, w, o), lambda: operators.grouped_gated_linear(x, w, w, o), lambda: operators.combine(x, o.view(1, 3)),
                 lambda: operators.grouped_linear_backward(x, x, w, o), lambda: operators.route_backward(x, x, o), lambda: operators.combine_backward(x, x, o, None, o)):
        with pytest.raises(ValueError, match="lives on cpu"):
            call()
    with pytest.raises(ValueError, match="holds torch.int32"):
        operators.route(x.int(), 2)
    with pytest.raises(ValueError, match="holds torch.float32"):
        operators.grouped_linear(x.float(), w.float(), o)


@pytest.mark.gpu
def test_what_is_refused():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 8, 64), dtype=torch.bfloat16, device="cuda")
    o, h, rows = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    places, weights, f = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda"), torch.zeros((4, 10), device="cuda")
    x8, w8, one = x.to(F8), w.to(F8), torch.ones(4, device="cuda")
    refused = [
        (lambda: operators.route(f, 0), "k of 0"), (lambda: operators.route(f, 11), "k of 11"), (lambda: operators.route(torch.zeros((1, 40), device="cuda"), 17), "k of 17"),
        (lambda: operators.route(torch.zeros((1, 1025), device="cuda"), 2), "experts"), (lambda: operators.route(f.double(), 2), "logits holds"),
        (lambda: operators.route(f.t(), 2), "next to each other"),
        (lambda: operators.route_backward(weights, f, places.long()), "experts is"), (lambda: operators.route_backward(weights[:, :1], f, places), "dweights"),
        (lambda: operators.route_backward(weights.half(), f, places), "dweights"), (lambda: operators.route_backward(weights, f[:3], places), "experts is"),
        (lambda: operators.grouped_linear(x, w, o.long()), "offsets holds"), (lambda: operators.grouped_linear(x, w, o[:2]), "matrices"), (lambda: operators.grouped_linear(x, w[0], o), "matrices"),
        (lambda: operators.grouped_linear(x, w.half(), o), "weight holds"), (lambda: operators.grouped_linear(x, w[:, :, :32], o), "matrices"),
        (lambda: operators.grouped_linear(x, w, o, rows=rows.float()), "rows holds"), (lambda: operators.grouped_linear(x, w, o, rows=places), "one number"),
        (lambda: operators.grouped_linear(x8, w8, o), "scales belong"), (lambda: operators.grouped_linear(x8, w8, o, x_scale=one, weight_scale=one), "weight_scale"),
        (lambda: operators.grouped_linear(x, w, o, dtype=torch.float16), "results"), (lambda: operators.grouped_linear(x, w, o[:1]), "offsets are"),
        (lambda: operators.grouped_linear(x, torch.zeros((2, 12, 64), dtype=torch.bfloat16, device="cuda")[:, :8], o), "one stride"),
        (lambda: operators.grouped_gated_linear(x, w, w[:, :4], o), "up_weight"), (lambda: operators.grouped_gated_linear(x, w, w, o, activation="tanh"), "activation"),
        (lambda: operators.grouped_linear_backward(x, x, w, o), "dy"), (lambda: operators.grouped_linear_backward(h, x, w, o, rows=rows[:3]), "dy"),
        (lambda: operators.grouped_linear_backward(h, x8, w8, o), "x holds"), (lambda: operators.grouped_gated_linear_backward(h, x, w, w, h, x, o), "up holds"),
        (lambda: operators.combine(x, places.long()), "places holds"), (lambda: operators.combine(x, places, weights=weights[:, :1]), "weights is"),
        (lambda: operators.combine(x, places, residual=h), "residual has shape"), (lambda: operators.combine(x.float(), places), "x holds"), (lambda: operators.combine(x[None], places), "row for each place"),
        (lambda: operators.combine_backward(x, x, places, weights, rows[:3]), "rows are"), (lambda: operators.combine_backward(h, x, places, weights, rows), "dy has shape"),
        (lambda: operators.combine_backward(x, x, places, weights.half(), rows), "weights is"),
    ]
    for call, message in refused:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(ValueError, match="requires a gradient"):
        operators.grouped_linear(x, torch.nn.Parameter(w), o)


def test_what_the_c_abi_refuses(capfd):
    """A message on stderr, 1, and nothing launched: the calls return before they reach the device (addresses here are no memory)."""
    w = runtime.wrappers()
    p = 4096
    calls = [
        w.tiramisu_hip_route(p, p, p, p, p, p, 4, 1025, 2, 0, 1, 0), w.tiramisu_hip_route(p, p, p, p, p, p, 4, 8, 9, 0, 1, 0), w.tiramisu_hip_route(p, p, p, p, p, p, 4, 8, 0, 0, 1, 0),
        w.tiramisu_hip_route(p, p, p, p, p, p, 1 << 25, 8, 2, 0, 1, 0), w.tiramisu_hip_route(p, p, p, p, p, p, 4, 8, 2, 0, 1, 3), w.tiramisu_hip_route(p, p, p, None, p, p, 4, 8, 2, 0, 1, 0),
        w.tiramisu_hip_route(None, p, p, p, p, p, 4, 8, 2, 0, 1, 0), w.tiramisu_hip_route_backward(p, p, None, p, 4, 8, 2, 0, 1, 0),
        w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 8, 7, 2, 8, 8, 0, 0, 2, 2), w.tiramisu_hip_grouped_linear(p, p, None, None, None, None, p, 8, 8, 2, 8, 8, 0, 0, 2, 2),
        w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 8, 8, 1025, 8, 8, 0, 0, 2, 2), w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 8, 8, 0, 8, 8, 0, 0, 2, 2),
        w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 8, 8, 2, 8, 1 << 22, 0, 0, 2, 2), w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 8, 8, 2, 8, 8, 0, 0, 3, 2),
        w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 1 << 28, 1 << 28, 2, 1 << 9, 8, 0, 0, 2, 2),
        w.tiramisu_hip_grouped_gated_linear(p, p, p, p, None, None, None, None, p, p, None, 8, 8, 2, 8, 8, 0, 0, 0, 4, 2, 2),
        w.tiramisu_hip_grouped_linear_backward(p, p, p, p, None, p, p, 8, 8, 2, 8, 8, 0, 0, 0, 3), w.tiramisu_hip_grouped_linear_backward(p, p, p, p, None, p, p, 8, 8, 2, 8, 8, 7, 0, 0, 2),
        w.tiramisu_hip_grouped_linear_backward(None, p, p, p, None, p, p, 8, 8, 2, 8, 8, 0, 0, 0, 2),
        w.tiramisu_hip_grouped_gated_linear_backward(p, p, p, p, p, p, p, None, p, p, None, 8, 8, 2, 8, 8, 0, 0, 0, 0, 0, 0, 4, 2),
        w.tiramisu_hip_grouped_gated_linear_backward(p, p, p, p, p, p, p, None, p, p, p, 8, 8, 2, 8, 8, 0, 0, 0, 7, 0, 0, 4, 2),
        w.tiramisu_hip_combine_rows(p, p, None, None, p, 4, 1025, 8, 8, 0, 0, 2), w.tiramisu_hip_combine_rows(p, p, None, None, p, 4, 2, 8, 8, 0, 0, 0),
        w.tiramisu_hip_combine_rows(p, None, None, None, p, 4, 2, 8, 8, 0, 0, 2), w.tiramisu_hip_combine_rows_backward(p, p, p, p, None, p, p, 4, 2, 8, 8, 0, 0, 2),
        w.tiramisu_hip_combine_rows_backward(p, p, p, None, p, p, p, 4, 2, 8, 8, 0, 0, 2), w.tiramisu_hip_combine_rows_backward(p, p, p, p, p, p, p, 1 << 25, 2, 8, 8, 0, 0, 2),
    ]
    assert calls == [1] * len(calls)
    messages = capfd.readouterr().err.strip().splitlines()
    assert len(messages) == len(calls) and all(m.startswith("Error at tiramisu_hip_") for m in messages)


def test_the_c_abi_refuses_sizes_that_pass_64_bits(capfd):
    w, p = runtime.wrappers(), 4096
    calls = [w.tiramisu_hip_grouped_gated_linear(p, p, p, p, None, None, None, None, p, None, None, 8, 8, 2, n, 8, 0, 0, 0, 4, 2, 2) for n in (1 << 63, (1 << 63) + 4, (1 << 64) - 1)]
    calls += [w.tiramisu_hip_grouped_gated_linear_backward(p, p, p, p, p, p, p, None, p, p, p, 8, 8, 2, 1 << 63, 8, 0, 0, 0, 0, 0, 0, 4, 2), w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, 1 << 63, 1 << 63, 2, 8, 8, 0, 0, 2, 2),
              w.tiramisu_hip_combine_rows(p, p, None, None, p, 1 << 63, 2, 8, 8, 0, 0, 2), w.tiramisu_hip_combine_rows_backward(p, p, p, p, p, p, p, 1 << 63, 2, 8, 8, 0, 0, 2)]
    assert calls == [1] * len(calls)
    assert len(capfd.readouterr().err.strip().splitlines()) == len(calls)


def test_the_c_abi_refuses_more_workgroups_than_a_launch_holds(capfd):
    w, p = runtime.wrappers(), 4096
    calls = [w.tiramisu_hip_combine_rows_backward(p, p, p, p, p, p, p, 4, 2, (1 << 30) - 1, 8, 0, 0, 2)]
    assert calls == [1] * len(calls)
    assert len(capfd.readouterr().err.strip().splitlines()) == len(calls)


def test_gradients_of_combine_without_columns_or_without_a_result():
    """Places are read wherever something is launched, also of rows without columns: without them such a call is refused.  Where no result is wanted, nothing is launched."""
    out = host_runtime.printed(r"""
p = 1 << 20
def says(*a):
    rc = w.tiramisu_hip_combine_rows_backward(*a, 0, 0, 2)
    return rc, len(launches())
# dy, x, places, owners, weights, dx, dweights, tokens, k, rows, columns
assert says(p, p, None, p, p, p, p, 4, 2, 8, 0) == (1, 0)
assert says(None, None, None, None, p, None, p, 4, 2, 0, 0) == (1, 0)
assert says(p, p, None, p, p, p, p, 4, 2, 8, 8) == (1, 0)
assert says(p, p, p, p, p, p, p, 4, 2, 8, 0) == (0, 1)
assert says(p, p, p, p, p, None, None, 4, 2, 8, 8) == (0, 0)
assert says(p, p, p, p, p, p, None, 4, 2, 8, 0) == (0, 0)
assert says(None, None, None, None, p, None, p, 4, 0, 0, 8) == (0, 0)
""")
    assert out == ""


# sizes of all groups, the share of them, places behind the last, N, K: few rows and tiles, shares that begin with empty groups, that are empty, that are all
SHARES = [([3, 0, 2, 1, 4, 0, 2, 1], 2, 5, 1, 70, 64), ([2] * 9, 8, 9, 0, 33, 40), ([1] * 20, 0, 20, 2, 20, 24), ([130, 7, 0, 300, 70, 1], 1, 3, 5, 130, 72), ([130, 7, 0, 300, 70, 1], 3, 6, 0, 264, 200),
          ([600, 520, 0, 700], 2, 3, 9, 300, 136), ([70, 300], 1, 2, 0, 1, 33), ([5000, 3, 2000, 900], 1, 4, 40, 300, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("sizes,low,high,behind,N,K", SHARES)
def test_some_of_the_groups(sizes, low, high, behind, N, K, dtype):
    """A share of the experts: its own offsets and weights with the places of all.  The others' places are rows of zeros, whatever the operands hold there."""
    out = torch.float16 if dtype == torch.float16 else torch.bfloat16
    share, S = slice(low, high), sum(sizes) + behind
    mine = torch.zeros((S, 1), dtype=torch.bool, device="cuda")
    mine[sum(sizes[:low]):sum(sizes[:high])] = True

    def zeros_elsewhere(got, name):
        assert not bool(got.masked_fill(mine, 0).any()), name

    for picked in (False, True):
        offsets, rows, x, xs, ws, scales, xd, wds = grouped_inputs(sizes, behind, N, K, dtype, 101 + N, weights=2, picked=picked)
        if not picked and dtype != F8:
            x = torch.where(mine, x, math.nan)
        own = offsets[low:high + 1]
        z = [torch.where(mine, by_group(sizes, behind, xd, wd, product), 0.0) for wd in wds]
        error = [sum_error(K, by_group(sizes, behind, xd, wd, sizes_of)) + by_group(sizes, behind, xd, wd, cut(dtype)) for wd in wds]
        for _ in range(2):
            torch.full((S, N), math.nan, device="cuda", dtype=out)          # (what the allocator hands out next)
            y = operators.grouped_linear(x, ws[0][share], own, rows=rows, x_scale=xs, weight_scale=None if xs is None else scales[0][share], dtype=out)
            zeros_elsewhere(y, "y")
            close(y, z[0], rounded(z[0], error[0], out), "y")
        unwritten = [torch.full((S, N), math.nan, device="cuda", dtype=out) for _ in range(3)]
        del unwritten
        got = operators.grouped_gated_linear(x, ws[0][share], ws[1][share], own, rows=rows, x_scale=xs, gate_scale=None if xs is None else scales[0][share],
                                             up_scale=None if xs is None else scales[1][share], dtype=out, keep_pre=True)
        for t, exact, bound, name in ((got.gate, z[0], error[0], "gate"), (got.up, z[1], error[1], "up")):
            zeros_elsewhere(t, name)
            close(t, exact, rounded(exact, bound, out), name)
        zeros_elsewhere(got.h, "h")
        assert bool(torch.isfinite(got.h.float()).all())
        if dtype == F8:
            continue
        g = generator(103)
        dy, gate, up = [torch.where(mine, normal((S, N), dtype, g), math.nan) for _ in range(3)]
        d = torch.where(mine, dy, 0).double()
        at = [sum(sizes[:e]) for e in range(low, high)]
        spans = [slice(a, a + n) for a, n in zip(at, sizes[low:high])]
        most = max(sizes[low:high])
        for _ in range(2):
            torch.full((S, K), math.nan, device="cuda", dtype=dtype)
            back = operators.grouped_linear_backward(dy, x, ws[0][share], own, rows=rows)
            zeros_elsewhere(back.dx, "dx")
            exact = by_group(sizes, behind, d, wds[0], lambda a, w: a @ w)
            close(back.dx, exact, backward_bound(dtype, exact, N, by_group(sizes, behind, d.abs(), wds[0].abs(), lambda a, w: a @ w)) + torch.zeros_like(exact), "dx")
            exact = torch.stack([d[s].t() @ xd[s] for s in spans])
            close(back.dweight, exact, backward_bound(dtype, exact, most, torch.stack([d[s].abs().t() @ xd[s].abs() for s in spans])), "dweight")
        both = operators.grouped_gated_linear_backward(dy, x, ws[0][share], ws[1][share], gate, up, own, rows=rows)
        zeros_elsewhere(both.dx, "gated dx")
        assert all(bool(torch.isfinite(t.float()).all()) for t in both)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES + [F8])
@pytest.mark.parametrize("sizes,behind,N,K", [([2, 0, 1, 3], 2, 70, 64), ([1] * 20, 3, 2100, 330), ([30, 0, 9], 20, 33, 70), ([40, 30], 9, 66, 71), ([130, 0, 60, 4], 30, 140, 200), ([700, 520, 3], 5, 264, 136),
                                              ([2600, 100, 1400], 100, 1104, 132), ([5000, 10, 3000], 50, 640, 264)])
def test_rows_that_are_none_of_x_are_zeros_whatever_the_weights_hold(sizes, behind, N, K, dtype):
    """Infinities and NaN in weights and in their scales do not reach places that take no row of x, nor those behind the groups: few rows, all tiles, rows moved ahead of them."""
    offsets, rows, x, xs, ws, scales, _, _ = grouped_inputs(sizes, behind, N, K, dtype, 107, weights=2, picked=True)
    T, S = x.shape[0], sum(sizes) + behind
    nobody = ~((rows >= 0) & (rows < T))
    nobody[sum(sizes):] = True
    assert int(nobody.sum()) > behind
    for w in ws:
        w[:, 0, 0] = math.nan
        w[:, N // 2, K - 1] = math.nan if dtype == F8 else math.inf
        w[0] = math.nan
    for s in scales:
        if s is not None:
            s[:, 1], s[0] = math.inf, math.nan
    odd = torch.zeros((T, K + 3), device="cuda").to(dtype)                  # rows at odd elements: moved ahead of tiles
    odd[:, 1:K + 1] = x
    for view in (x, odd[:, 1:K + 1]):
        y = operators.grouped_linear(view, ws[0], offsets, rows=rows, x_scale=xs, weight_scale=scales[0])
        assert y.shape == (S, N) and not bool(y[nobody].any()) and bool(torch.isnan(y[~nobody][:, 0]).all())
        for activation in ("silu", "gelu"):
            got = operators.grouped_gated_linear(view, ws[0], ws[1], offsets, rows=rows, activation=activation, x_scale=xs, gate_scale=scales[0], up_scale=scales[1], keep_pre=True)
            assert not any(bool(t[nobody].any()) for t in got) and all(bool(torch.isnan(t[~nobody][:, 0]).all()) for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(1025, 8195), (1024, 8191)])
def test_gradients_of_weights_around_the_size_that_goes_past_the_caches(N, K):
    """2^27 bytes of eight groups' gradients and some less or more, rows at odd elements; terms of a tile shared among workgroups or not."""
    dtype, sizes = torch.bfloat16, [70, 0, 3, 130, 1, 0, 40, 9]
    offsets, _, x, _, (w,), _, xd, _ = grouped_inputs(sizes, 5, N, K, dtype, 127)
    dy = normal((x.shape[0], N), dtype, generator(131))
    got, d, at = operators.grouped_linear_backward(dy, x, w, offsets).dweight, dy.double(), 0
    for e, n in enumerate(sizes):
        a, b = d[at:at + n].t(), xd[at:at + n]
        at += n
        close(got[e], a @ b, backward_bound(dtype, a @ b, n, a.abs() @ b.abs()), "group %d" % e)
