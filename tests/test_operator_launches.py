"""Every way in which the operators' products are launched, against their definitions in 64 bits: one ragged size for each tile, each split of k, both gradients in one
launch and in two.  That a size takes the way it is here for, and that all kernels are launched by some size, is checked on the host (host_runtime.py)."""
import json

import pytest
import torch

import host_runtime
import test_operators as definitions
from tiramisu_amd import operators, runtime

F8 = torch.float8_e4m3fn
HALVES = [torch.bfloat16, torch.float16]

# launches: (M, N, K).  N and M odd, K no multiple of a slice.
LINEAR_16 = {
    "few": (9, 93, 330), "few, 32": (31, 61, 166), "few, 64": (53, 45, 234),
    "y 64x64": (143, 9, 46), "y 64x64 split": (65, 9, 2918), "y 128x64": (135, 5677, 44), "y 128x64 split": (2267, 9, 4028), "y 128x128": (3965, 513, 32),
    "y 256x128": (3311, 1369, 34), "y 256x256": (3661, 3551, 146), "y 128x128 split": (145, 2743, 5258), "y 256x128 split": (6931, 69, 11422), "y 256x256 split": (521, 3609, 11362),
}
LINEAR_8 = {
    "few": (9, 93, 332), "few, 32": (31, 61, 164), "few, 64": (53, 45, 236),
    "y 64x64": (143, 9, 44), "y 128x64": (147, 5807, 36), "y 128x128": (331, 5645, 644), "y 256x128": (1655, 3815, 292), "y 256x256": (2805, 4937, 284),
    "y 64x64 split": (1, 9, 28264), "y 128x64 split": (2823, 9, 10444), "y 256x128 split": (5011, 427, 12796),
}
GATED_16 = {
    "few": (9, 93, 330), "few, 32": (31, 61, 166), "few, 64": (53, 45, 234),
    "y 64x128": (79, 9, 36), "y 64x128 split": (15, 9, 3982), "y 128x128": (131, 5649, 34), "y 128x128 split": (3527, 9, 2834), "y 256x128": (1655, 2059, 34),
    "y 256x256": (1113, 5619, 136), "y 256x128 split": (9391, 9, 3784), "y 256x256 split": (141, 6435, 12082),
}
GATED_8 = {
    "few": (9, 93, 332), "few, 32": (31, 61, 164), "few, 64": (53, 45, 236),
    "y 64x128": (67, 9, 36), "y 128x128": (1633, 635, 1232), "y 256x128": (981, 3487, 560), "y 256x256": (2771, 2693, 420),
    "y 64x128 split": (1, 11, 12400), "y 256x128 split": (6315, 149, 12104),
}
LINEAR_BACKWARD = {
    "dx and dw 64x64": (1, 11, 34), "dw and dx 64x64": (67, 9, 34), "dx and dw 128x64": (65, 133, 3436), "dw and dx 128x64": (143, 65, 3758), "dx and dw 128x128": (327, 365, 2830),
    "dw and dx 128x128": (371, 279, 3688), "dx and dw 256x128": (657, 795, 3736), "dw and dx 256x128": (875, 769, 2744), "dx and dw 256x256": (1237, 1461, 3468),
    "dw and dx 256x256": (2419, 2251, 2040),
    "dx 64x64, dw 64x64 split": (3733, 11, 34), "dx 64x64 split, dw 64x64": (1, 3991, 34), "dx 64x64 split, dw 128x64": (1, 6079, 132), "dx 64x64 split, dw 128x128": (1, 5897, 344),
    "dx 64x64 split, dw 256x128": (1, 5517, 850), "dx 128x64 split, dw 64x64": (1155, 5751, 66), "dx 128x64, dw 128x128": (1191, 1685, 1474), "dx 128x128, dw 128x64": (1715, 1043, 1770),
    "dx 128x128, dw 256x128": (957, 1233, 3718), "dx 128x64, dw 256x256": (315, 3707, 4058), "dx 256x128, dw 128x128": (1419, 987, 3986), "dx 256x256, dw 128x64": (3327, 419, 4038),
    "dx 128x128 split, dw 128x128": (73, 10085, 4168), "dx 256x128 split, dw 128x128": (151, 14655, 2786), "dx 256x256 split, dw 256x256": (823, 14315, 2882),
    "dx 128x128, dw 128x64 split": (9009, 71, 1156), "dx 256x256, dw 128x128 split": (8139, 67, 5974), "dx 256x256, dw 256x128 split": (8231, 129, 5790),
    "dx 256x256, dw 256x256 split": (17381, 519, 3916),
}
GATED_BACKWARD = {
    "dx and dw 64x64": (1, 9, 50), "dw and dx 64x64": (81, 11, 32), "dx and dw 128x64": (71, 53, 4164), "dw and dx 128x64": (135, 33, 3824), "dx and dw 128x128": (249, 147, 3976),
    "dw and dx 128x128": (565, 255, 2008), "dx and dw 256x128": (747, 435, 2750), "dw and dx 256x128": (705, 335, 2936), "dx and dw 256x256": (1087, 583, 3810),
    "dw and dx 256x256": (1915, 891, 2576),
    "dx 64x64, dw 64x64 split": (3901, 9, 34), "dx 64x64 split, dw 64x64": (1, 1881, 42), "dx 64x64 split, dw 256x128": (1, 3627, 532), "dx 128x64 split, dw 128x64 split": (4157, 4759, 36),
    "dx 128x64 split, dw 128x128": (65, 4897, 1022), "dx 128x64 split, dw 256x256": (181, 5537, 1274), "dx 128x64, dw 128x128": (1523, 1345, 1194), "dx 128x128 split, dw 128x128": (129, 5591, 3114),
    "dx 128x128, dw 128x64": (1479, 519, 1724), "dx 256x128 split, dw 256x256": (1195, 4197, 1744), "dx 256x128, dw 64x64": (2581, 409, 2358), "dx 256x256, dw 128x128": (3979, 547, 3256),
    "dx 256x256, dw 256x128": (3191, 687, 3902), "dx 256x256 split, dw 256x256": (131, 9765, 8252), "dx 128x128, dw 128x128 split": (17879, 1369, 66),
    "dx 128x128, dw 256x128 split": (20999, 2103, 74), "dx 256x256, dw 256x256 split": (15271, 305, 4314),
}
# rows, columns: what definitions.test_norm_backward leaves out, and rows that teams take several of
NORM_BACKWARD = [(40, 400), (600, 1001), (5000, 2001), (900, 3999)]


def sizes(table):
    return sorted(set(table.values()))


def test_each_size_takes_its_launches_and_all_kernels_are_launched():
    def shapes(test):
        return [m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0] == "rows,columns"][0]

    out = host_runtime.printed("""
import json, re
p = 1 << 20
LAYOUT = {("1", "1"): "y", ("1", "0"): "dx", ("0", "0"): "dw"}
used = set()
def described():
    parts = []
    for k, b, t in launches():
        used.add(k)
        c = [(LAYOUT[g[2:]], "%%sx%%s" %% g[:2]) for g in re.findall(r"ILi\\d+ELi(\\d+)ELi(\\d+)ELi\\d+ELi\\d+ELi\\d+ELb(\\d)ELb(\\d)E", k)]
        if "pair" in k: parts.append("%%s and %%s %%s" %% (c[0][0], "dw" if c[0][0] == "dx" else "dx", c[0][1]))
        elif c: parts.append("%%s %%s" %% c[0])
        elif "few" in k: parts.append("few")
        elif "finish" in k: parts[-1] += " split"
    return ", ".join(parts)
linear_16, linear_8, gated_16, gated_8, linear_backward, gated_backward, norms, norms_backward = json.loads(%r)
def say(kind, table, call):
    for name, size in table.items():
        assert call(*size) == 0
        got = described()
        if got != name.split(", 32")[0].split(", 64")[0]: print("%%s %%s: %%s, not %%s" %% (kind, size, got, name))
    w.tiramisu_hip_release_cached_memory()
for t in (1, 2):
    say("linear", linear_16, lambda M, N, K: w.tiramisu_hip_linear(p, p, p, p, None, None, p, p, M, N, K, 0, 0, 0, 0, t, t))
    say("linear, 8 bits", linear_8, lambda M, N, K: w.tiramisu_hip_linear(p, p, p, p, p, p, p, p, M, N, K, 0, 0, 0, 0, 3, t))
    say("gated", gated_16, lambda M, N, K: w.tiramisu_hip_gated_linear(p, p, p, None, None, None, p, p, p, M, N, K, 0, 0, 0, 4, t, t))
    say("gated, 8 bits", gated_8, lambda M, N, K: w.tiramisu_hip_gated_linear(p, p, p, p, p, p, p, p, p, M, N, K, 0, 0, 0, 4, 3, t))
    say("linear backward", linear_backward, lambda M, N, K: w.tiramisu_hip_linear_backward(p, p, p, p, p, p, p, M, N, K, 0, 0, 0, 0, 2, t))
    say("gated backward", gated_backward, lambda M, N, K: w.tiramisu_hip_gated_linear_backward(p, p, p, p, p, p, p, p, p, M, N, K, 0, 0, 0, 0, 0, 0, 4, t))
# rows at odd elements, moved ahead of the tiles, are in definitions.test_operands_within_larger_tensors
w.tiramisu_hip_linear(p + 2, p, None, None, None, None, p, None, 300, 260, 100, 0, 0, 0, 0, 2, 2)
w.tiramisu_hip_linear(p + 1, p, None, None, p, p, p, None, 300, 260, 100, 0, 0, 0, 0, 3, 2)
for t in (0, 1, 2):
    for rows, columns in norms:
        w.tiramisu_hip_rms_norm(p, None, p, p, None, None, p, rows, columns, 0, 0, 1e-6, t, t)
        w.tiramisu_hip_rms_norm(p, None, p, p, None, p, p, rows, columns, 0, 0, 1e-6, t, 3)
    for rows, columns in norms_backward:
        w.tiramisu_hip_rms_norm_backward(p, p, p, p, None, p, p, rows, columns, 0, 0, 0, t)
described()
for k in sorted(set(k for k in hip.recording_kernels().decode().split() if k.startswith("_ZN4tops")) - used): print("never launched:", k)
""" % json.dumps([LINEAR_16, LINEAR_8, GATED_16, GATED_8, LINEAR_BACKWARD, GATED_BACKWARD, shapes(definitions.test_norm), shapes(definitions.test_norm_backward) + NORM_BACKWARD]))
    assert out == "", out


# ---------------------------------------------------------------- forward

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out,M,N,K", [(d, d, *size) for d in HALVES for size in sizes(LINEAR_16)] + [(F8, d, *size) for d in HALVES for size in sizes(LINEAR_8)])
def test_linear(M, N, K, dtype, out):
    """Bias, residual and the sums ahead of the activation in all combinations, with and without an activation."""
    x, xs, (w,), (ws,), xd, (wd,) = definitions.product_inputs(M, N, K, dtype, M + N + K)
    g = definitions.generator(107)
    bias, residual = definitions.normal((N,), out, g), definitions.normal((M, N), out, g)
    z, size, cut = xd @ wd.t(), xd.abs() @ wd.abs().t(), definitions.cut_off(xd, wd, dtype)
    for case in range(16):
        b, r, keep, activation = bias if case & 1 else None, residual if case & 2 else None, bool(case & 4), "gelu" if case & 8 else "none"
        got = operators.linear(x, w, bias=b, residual=r, activation=activation, x_scale=xs, weight_scale=ws, dtype=out, keep_pre=keep)
        pre = z if b is None else z + b.double()
        error = definitions.sum_error(K, size if b is None else size + b.double().abs()) + cut
        y = definitions.exact_activation(activation, pre)
        slack = pre.abs() + 1
        if r is not None:
            y, slack = y + r.double(), slack + r.double().abs()
        what = "%s%s%s" % (activation, ", bias" if b is not None else "", ", residual" if r is not None else "")
        definitions.close(got.y, y, definitions.rounded(y, 1.13 * error + 2.0 ** -22 * slack, out), what)
        assert got.y.dtype == out and (got.pre is not None) == keep
        if keep:
            definitions.close(got.pre, pre, definitions.rounded(pre, error, out), what + ": pre")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,M,N,K", [(d, *size) for d in HALVES for size in sizes(GATED_16)] + [(F8, *size) for size in sizes(GATED_8)])
def test_gated_linear(M, N, K, dtype):
    definitions.test_gated_linear(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", sizes(GATED_8))
def test_gated_linear_of_8_bits_in_float16(M, N, K):
    x, xs, ws, scales, xd, (gd, ud) = definitions.product_inputs(M, N, K, F8, 109, weights=2)
    got = operators.gated_linear(x, ws[0], ws[1], x_scale=xs, gate_scale=scales[0], up_scale=scales[1], dtype=torch.float16, keep_pre=True)
    for out, wd in ((got.gate, gd), (got.up, ud)):
        exact = xd @ wd.t()
        definitions.close(out, exact, definitions.rounded(exact, definitions.sum_error(K, xd.abs() @ wd.abs().t()) + definitions.cut_off(xd, wd, F8), torch.float16), "a projection")
    # h of the projections as they are kept: each is off by its rounding, 2^-11, silu's slope is 1.1 at most
    gate, up = got.gate.double(), got.up.double()
    a = definitions.exact_activation("silu", gate)
    u = definitions.ROUNDOFF[torch.float16] * 1.01
    bound = 1.13 * (u * gate.abs() + 2.0 ** -24) * up.abs() * 1.01 + a.abs() * (u * up.abs() + 2.0 ** -24) + 2.0 ** -22 * (gate.abs() + 1) * up.abs()
    definitions.close(got.h, a * up, definitions.rounded(a * up, bound, torch.float16), "h")


# ---------------------------------------------------------------- backward

@pytest.fixture(autouse=True)
def slope_of_relu_at_zero(monkeypatch):
    """It is 0.  Autograd's slope of a clamp is 1 there, which only sizes like these show: among a million normal numbers in 16 bits some are zero."""
    slope = definitions.exact_slope
    monkeypatch.setattr(definitions, "exact_slope", lambda name, z: (z > 0).double() if name == "relu" else slope(name, z))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
@pytest.mark.parametrize("rows,columns", NORM_BACKWARD)
def test_norm_backward(rows, columns, dtype):
    definitions.test_norm_backward(rows, columns, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", sizes(LINEAR_BACKWARD))
def test_linear_backward(M, N, K, dtype):
    definitions.test_linear_backward(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", sizes(GATED_BACKWARD))
def test_gated_linear_backward(M, N, K, dtype):
    definitions.test_gated_linear_backward(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(65, 133, 346), (3733, 11, 34), (1, 3991, 34)])
def test_gradients_that_are_not_asked_for(M, N, K):
    """From C each gradient may be left out: the others are what they are with it, within the rounding of their sums' order."""
    w = runtime.wrappers()
    g = definitions.generator(113)
    dy, x, weight, up = [definitions.normal(shape, torch.bfloat16, g) for shape in ((M, N), (M, K), (N, K), (N, K))]
    pre, gate, kept_up = [definitions.normal((M, N), torch.bfloat16, g) for _ in range(3)]
    whole = operators.linear_backward(dy, x, weight, pre=pre, activation="silu", bias=True)
    whole_gated = operators.gated_linear_backward(dy, x, weight, up, gate, kept_up)
    torch.cuda.synchronize()
    before = w.tiramisu_hip_get_stream()
    w.tiramisu_hip_set_stream(w.tiramisu_hip_null_stream())
    try:
        for asked in range(8):
            out = [torch.full_like(t, 7.0) for t in whole]
            at = [t.data_ptr() if asked >> i & 1 else None for i, t in enumerate(out)]
            assert w.tiramisu_hip_linear_backward(dy.data_ptr(), x.data_ptr(), weight.data_ptr(), pre.data_ptr(), *at, M, N, K, 0, 0, 0, 0, 4, 2) == 0
            for i, (got, was) in enumerate(zip(out, whole)):
                assert bool((got == 7.0).all()) if not asked >> i & 1 else float((got.float() - was.float()).abs().max()) <= 2.0 ** -7 * float(was.float().abs().max())
        for asked in range(4):
            out = [torch.full_like(t, 7.0) for t in whole_gated]
            at = [t.data_ptr() if asked >> min(i, 1) & 1 else None for i, t in enumerate(out)]
            assert w.tiramisu_hip_gated_linear_backward(dy.data_ptr(), x.data_ptr(), weight.data_ptr(), up.data_ptr(), gate.data_ptr(), kept_up.data_ptr(), *at, M, N, K,
                                                        0, 0, 0, 0, 0, 0, 4, 2) == 0
            for i, (got, was) in enumerate(zip(out, whole_gated)):
                assert bool((got == 7.0).all()) if not asked >> min(i, 1) & 1 else float((got.float() - was.float()).abs().max()) <= 2.0 ** -7 * float(was.float().abs().max())
    finally:
        w.tiramisu_hip_set_stream(before)
        torch.cuda.synchronize()
