"""Every way in which the operators of experts and of 4-bit weights are launched, against their definitions in 64 bits: one ragged size for each tile, each number of wavefronts that share k, each
width of a router.  That a size takes the way it is here for, and that all kernels are launched by some size, is checked on the host (host_runtime.py)."""
import json
import random

import pytest
import torch

import host_runtime
import test_expert_operators as experts
import test_four_bit as four_bit
from test_operators import F8, HALVES

# launches: (rows, groups, N, K)
LINEAR_16 = {"few 8": (30, 19, 93, 330), "few 4": (16, 8, 2100, 1030), "few 2": (20, 9, 4100, 330), "64x64/3": (83, 3, 93, 142), "128x128/4": (418, 117, 67, 42), "128x128/2": (164, 52, 815, 38),
             "256x128/3": (29169, 23, 67, 134), "256x256/2": (5294, 25, 1601, 162), "192x128/2": (5929, 11, 1026, 142)}
GATED_16 = {"few 8": (30, 19, 93, 330), "few 4": (16, 8, 2100, 330), "64x128/3": (83, 3, 93, 142), "128x128/4": (40, 3, 93, 42), "128x128/2": (24628, 82, 9, 38), "256x128/3": (32239, 2, 9, 158),
            "256x256/2": (18525, 77, 205, 154), "192x128/2": (2853, 9, 1104, 132)}
LINEAR_8 = {"few 8": (30, 19, 93, 332), "few 4": (16, 8, 2100, 3000), "few 2": (20, 9, 4100, 332), "64x64/3": (83, 3, 93, 140), "128x128/4": (250, 8, 2029, 392), "256x128/3": (36058, 51, 71, 44),
            "256x256/2": (30200, 22, 235, 36)}
GATED_8 = {"few 8": (30, 19, 93, 332), "few 4": (16, 8, 2100, 332), "64x128/3": (83, 3, 93, 140), "128x128/4": (14642, 11, 13, 36), "256x128/3": (28360, 65, 9, 820), "256x256/2": (11240, 4, 617, 36)}
LINEAR_BACKWARD = {"64x64/3": (130, 9, 12, 34), "128x128/2": (103, 112, 14, 74), "128x128/4": (101, 21, 12, 446), "256x128/3": (4599, 96, 202, 78), "256x256/2": (3277, 30, 134, 986),
                   "64x64/3 split": (1125, 1, 12, 34), "128x128/2 split": (12152, 4, 10, 38), "128x128/4 split": (6115, 3, 12, 74), "256x128/3 split": (11936, 1, 1416, 66), "256x256/2 split": (20158, 1, 132, 2098)}
GATED_BACKWARD = {"64x64/3": (130, 9, 11, 34), "128x128/2": (103, 112, 13, 74), "128x128/4": (101, 21, 11, 446), "256x128/3": (3520, 105, 113, 82), "256x256/2": (4001, 13, 1130, 1026),
                  "64x64/3 split": (1125, 1, 11, 34), "128x128/2 split": (12152, 4, 9, 38), "128x128/4 split": (6115, 3, 11, 74), "256x128/3 split": (13090, 1, 787, 74), "256x256/2 split": (23260, 1, 99, 1134)}
# (M, N, K): k in several chunks of LDS and behind their last whole unit
FOUR_BIT = {"few 1 8": (5, 100, 4330), "few 1 4": (9, 4203, 330), "few 2 8": (20, 100, 2330), "few 2 4": (31, 4203, 331), "few 2 2": (17, 8301, 200), "few 4 8": (50, 100, 2330), "few 4 4": (64, 4203, 130),
            "few 4 2": (33, 8301, 1290), "few 4 8, in parts": (130, 100, 500), "widened": (3001, 700, 1333)}
FOUR_BIT_GATED = {"few 1 8": (5, 100, 4330), "few 1 4": (9, 4203, 330), "few 2 8": (20, 100, 2330), "few 2 4": (31, 4203, 331), "few 4 8": (50, 100, 2330), "few 4 4": (64, 8301, 130), "widened": (3001, 700, 1333)}
# tokens, experts, k
ROUTES = [(tokens, count, k) for tokens in (9, 300) for count, k in ((9, 2), (25, 3), (50, 16), (120, 4), (250, 4), (500, 5), (900, 3))]


def sizes(table):
    return sorted(set(table.values()))


def test_each_size_takes_its_launch_and_all_kernels_are_launched():
    out = host_runtime.printed(r"""
import json, re
p = 1 << 20
used = set()
def described():
    parts = []
    for k, b, t in launches():
        used.add(k)
        c = re.findall(r"ILi\d+ELi(\d+)ELi(\d+)ELi\d+ELi\d+ELi(\d+)ELb", k)
        few = re.search(r"grouped_few_kernelI(?:Li\d+E){4}Li(\d)E", k)
        bits = re.search(r"four_bit_few_kernelILi\d+ELi\d+ELi(\d)ELi(\d)E", k)
        if few: parts.append("few " + few[1])
        elif bits: parts.append("few %%s %%s" %% bits.groups())
        elif "widen" in k and "widened" not in parts: parts.append("widened")
        elif c and "tgroups" in k: parts.append("%%sx%%s/%%s" %% c[0])
        elif "weights_finish" in k: parts[-1] += " split"
    return ", ".join(parts)
tables = json.loads(%r)
def say(kind, table, call):
    for name, size in tables[table].items():
        assert call(*size) == 0
        got = described()
        if got != name.replace(", in parts", ""): print("%%s %%s: %%s, not %%s" %% (kind, size, got, name))
    w.tiramisu_hip_release_cached_memory()
for t in (1, 2):
    say("linear", "linear_16", lambda S, E, N, K: w.tiramisu_hip_grouped_linear(p, p, p, None, None, None, p, S, S, E, N, K, 0, 0, t, t))
    say("linear, 8 bits", "linear_8", lambda S, E, N, K: w.tiramisu_hip_grouped_linear(p, p, p, None, p, p, p, S, S, E, N, K, 0, 0, 3, t))
    say("gated", "gated_16", lambda S, E, N, K: w.tiramisu_hip_grouped_gated_linear(p, p, p, p, None, None, None, None, p, p, p, S, S, E, N, K, 0, 0, 0, 4, t, t))
    say("gated, 8 bits", "gated_8", lambda S, E, N, K: w.tiramisu_hip_grouped_gated_linear(p, p, p, p, None, p, p, p, p, p, p, S, S, E, N, K, 0, 0, 0, 4, 3, t))
    say("linear backward", "linear_backward", lambda S, E, N, K: w.tiramisu_hip_grouped_linear_backward(p, p, p, p, None, p, p, S, S, E, N, K, 0, 0, 0, t))
    say("gated backward", "gated_backward", lambda S, E, N, K: w.tiramisu_hip_grouped_gated_linear_backward(p, p, p, p, p, p, p, None, p, p, p, S, S, E, N, K, 0, 0, 0, 0, 0, 0, 4, t))
    say("4 bits", "four_bit", lambda M, N, K: w.tiramisu_hip_four_bit_linear(p, p, p, p, p, p, M, N, K, 0, 0, 0, 0, 2, t))
    say("4 bits, gated", "four_bit_gated", lambda M, N, K: w.tiramisu_hip_four_bit_gated_linear(p, p, p, p, p, p, M, N, K, 0, 0, 0, 0, 0, 4, t))
    for columns in (100, 1000):
        w.tiramisu_hip_combine_rows(p, p, p, p, p, 9, 2, 20, columns, 0, 0, t)
        w.tiramisu_hip_combine_rows_backward(p, p, p, p, p, p, p, 9, 2, 20, columns, 0, 0, t)
for t in (0, 1, 2):
    for tokens, count, k in tables["routes"]:
        w.tiramisu_hip_route(p, p, p, p, p, p, tokens, count, k, 0, 1, t)
        w.tiramisu_hip_route_backward(p, p, p, p, tokens, count, k, 0, 1, t)
    w.tiramisu_hip_quantize_groups(p, p, p, 4, 40, 0, t)
# rows at odd elements, moved ahead of the tiles, are in experts.test_grouped_operands_within_larger_tensors
w.tiramisu_hip_grouped_linear(p + 2, p, p, p, None, None, p, 300, 200, 3, 260, 100, 0, 0, 2, 2)
w.tiramisu_hip_grouped_linear(p + 1, p, p, p, p, p, p, 300, 200, 3, 260, 100, 0, 0, 3, 2)
described()
mine = ("_ZN7tgroups", "_ZN6troute", "_ZN8tcombine", "_ZN5tfour")
for k in sorted(set(k for k in hip.recording_kernels().decode().split() if k.startswith(mine)) - used): print("never launched:", k)
""" % json.dumps({"linear_16": LINEAR_16, "gated_16": GATED_16, "linear_8": LINEAR_8, "gated_8": GATED_8, "linear_backward": LINEAR_BACKWARD, "gated_backward": GATED_BACKWARD,
                  "four_bit": FOUR_BIT, "four_bit_gated": FOUR_BIT_GATED, "routes": ROUTES}))
    assert out == "", out


def spread(rows, groups):
    """Sizes of groups as routers leave them: uneven, some empty; and some rows behind the last."""
    rng = random.Random(rows + groups)
    behind = rows // 50
    liked = [rng.expovariate(1.0) if rng.random() < 0.9 else 0.0 for _ in range(groups - 1)] + [1.0]
    counts = [0] * groups
    for g in rng.choices(range(groups), liked, k=rows - behind):
        counts[g] += 1
    return counts, behind


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out,rows,groups,N,K", [(d, d, *s) for d in HALVES for s in sorted(set(sizes(LINEAR_16) + sizes(GATED_16)))] + [(F8, d, *s) for d in HALVES for s in sorted(set(sizes(LINEAR_8) + sizes(GATED_8)))])
def test_grouped(rows, groups, N, K, dtype, out):
    experts.check_grouped(*spread(rows, groups), N, K, dtype, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,groups,N,K", sorted(set(sizes(LINEAR_BACKWARD) + sizes(GATED_BACKWARD))))
def test_grouped_backward(rows, groups, N, K, dtype):
    experts.check_grouped_backward(*spread(rows, groups), N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_gradient_of_a_group_of_many_rows(dtype):
    """More rows than an index in LDS holds at a time, in one group of three."""
    experts.check_grouped_backward([9000, 0, 70], 30, 40, 72, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", sizes(FOUR_BIT))
def test_four_bit_linear(M, N, K, dtype):
    four_bit.test_four_bit_linear(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("M,N,K", sizes(FOUR_BIT_GATED))
def test_four_bit_gated_linear(M, N, K, dtype):
    four_bit.test_four_bit_gated_linear(M, N, K, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", experts.WIDE)
@pytest.mark.parametrize("tokens,count,k", ROUTES)
def test_route(tokens, count, k, dtype):
    experts.test_route(tokens, count, k, dtype)
    experts.test_route_backward(tokens, count, k, dtype)
