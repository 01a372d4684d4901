"""The operators of a feed-forward sublayer with experts and of one with 4-bit weights, as a program of their user runs them.

* route:   each token's k best experts by the router's logits, their weights, and the tokens' places grouped by expert; backward;
* grouped linear, grouped gated: matrix products of rows that are grouped by expert, every group with weights of its own, the groups of any size (a
           router's choice: most uneven, some empty); forward on 16 and 8 bits, backward, one token to a long prompt;
* combine: the weighted sum of a token's rows, added to the residual stream; backward;
* four-bit linear, four-bit gated: products of some tokens with weights in 4 bits (e2m1) and a power of two for each 32 of a row.

Weights are [outputs, inputs] or [experts, outputs, inputs], rows of x are tokens.  All tensors live on the GPU.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32, "float8": torch.float8_e4m3fn}
E4M3_MOST = 448.0
GROUP = 32                                                      # weights of a row that share a scale, in 4 bits
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # serving, one token: launches are all that it costs
        {"name": "route one token", "kind": "route", "tokens": 1, "experts": 64, "k": 8, "dtype": "bfloat16", "normalise": True, "padded": 0.0},
        # a long padded prompt through a 32-bit router: padding has no expert
        {"name": "route prompt", "kind": "route", "tokens": 16384, "experts": 128, "k": 8, "dtype": "float32", "normalise": True, "padded": 0.05},
        # serving, one token: the weights of the experts that it chose
        {"name": "experts one token", "kind": "grouped_gated", "tokens": 1, "experts": 64, "k": 8, "N": 1024, "K": 2048, "dtype": "bfloat16", "activation": "silu", "keep": False},
        # a long prompt through many small experts
        {"name": "experts prompt", "kind": "grouped_gated", "tokens": 4096, "experts": 64, "k": 8, "N": 1024, "K": 2048, "dtype": "bfloat16", "activation": "silu", "keep": False},
        # a ragged batch in 8 bits, at sizes that nothing divides
        {"name": "experts ragged 8 bits", "kind": "grouped_gated", "tokens": 1000, "experts": 12, "k": 2, "N": 1500, "K": 700, "dtype": "float8", "activation": "gelu", "keep": False},
        # training: gradients of the rows and of both weights of every expert
        {"name": "experts backward", "kind": "grouped_gated_backward", "tokens": 4096, "experts": 32, "k": 4, "N": 1024, "K": 2048, "dtype": "bfloat16", "activation": "silu"},
        # serving, sixteen sequences by a token each: the down projection, most experts with a row or two
        {"name": "experts down 16 tokens", "kind": "grouped_linear", "tokens": 16, "experts": 64, "k": 8, "N": 2048, "K": 1024, "dtype": "bfloat16"},
        # training at a size that no tile divides
        {"name": "experts down backward", "kind": "grouped_linear_backward", "tokens": 1500, "experts": 10, "k": 3, "N": 1000, "K": 700, "dtype": "float16"},
        # a long prompt's way back into the residual stream
        {"name": "combine prompt", "kind": "combine", "tokens": 4096, "k": 8, "N": 2048, "dtype": "bfloat16", "weights": True, "residual": True, "padded": 0.05},
        # training: gradients of the experts' rows and of the router's weights
        {"name": "combine backward", "kind": "combine_backward", "tokens": 2000, "k": 3, "N": 1430, "dtype": "float16", "padded": 0.0},
        # serving, one token: the output projection in 4 bits, bound by launches and the weights' bytes
        {"name": "4 bits one token", "kind": "four_bit", "M": 1, "N": 4096, "K": 4096, "dtype": "bfloat16", "activation": "none", "bias": False, "residual": True},
        # serving, sixteen sequences by a token each: both projections of a wide gated layer
        {"name": "4 bits gated 16 tokens", "kind": "four_bit_gated", "M": 16, "N": 8192, "K": 2048, "dtype": "bfloat16", "activation": "silu"},
    ]


def draw(rng):
    def size(low, high, step=1):
        """Spread over the logarithm; half of the sizes are what they are, half a multiple of `step`."""
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if step > 1 and rng.random() < 0.5:
            v = (v + step // 2) // step * step
        return max(low, min(high, v))

    kind = rng.choice(["route", "route_backward", "grouped_linear", "grouped_gated", "grouped_linear_backward", "grouped_gated_backward", "combine", "combine_backward", "four_bit",
                       "four_bit_gated"])
    half = rng.choice(["bfloat16", "float16"])
    if kind.startswith("route"):
        experts = size(2, 256, 8)
        return {"kind": kind, "tokens": size(1, 16384), "experts": experts, "k": rng.randint(1, min(8, experts)), "dtype": rng.choice(["bfloat16", "float16", "float32"]),
                "normalise": rng.random() < 0.6, "padded": rng.choice([0.0, 0.05])}
    if kind.startswith("combine"):
        k = rng.randint(1, 8)
        case = {"kind": kind, "tokens": size(1, 32768 // k), "k": k, "N": size(64, 2048, 64), "dtype": half, "padded": rng.choice([0.0, 0.05])}
        if kind == "combine":
            case.update(weights=rng.random() < 0.7, residual=rng.random() < 0.6)
        return case
    if kind.startswith("four_bit"):
        case = {"kind": kind, "M": rng.choice([size(1, 64), size(1, 2048, 16)]), "N": size(64, 8192, 64), "K": size(64, 4096, 64), "dtype": half,
                "activation": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"] if kind == "four_bit" else ["silu", "gelu", "gelu_tanh", "relu"])}
        if kind == "four_bit":
            case.update(bias=rng.random() < 0.5, residual=rng.random() < 0.5)
        return case
    experts = size(2, 64)
    k = rng.randint(1, min(8, experts))
    backward = kind.endswith("backward")
    case = {"kind": kind, "tokens": size(16 if backward else 1, (16384 if backward else 32768) // k), "experts": experts, "k": k, "N": size(64, 1024, 64), "K": size(64, 2048, 64),
            "dtype": half if backward else rng.choice([half, half, "float8"])}
    if "gated" in kind:
        case["activation"] = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
        if not backward:
            case["keep"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------- inputs

def _rows_in_8_bits(t):
    """What a program that serves in 8 bits keeps of a matrix: e4m3 values and one scale for each row."""
    scale = t.abs().amax(-1) / E4M3_MOST
    return (t / scale[..., None]).to(torch.float8_e4m3fn), scale


def _rows_in_4_bits(t):
    """... in 4 bits: e2m1 values, two to a byte (the first in the low half), and the exponent of a power of two for each 32 of a row."""
    rows, columns = t.shape
    t = torch.nn.functional.pad(t, (0, -columns % GROUP))
    groups = t.view(rows, -1, GROUP)
    exponent = torch.ceil(torch.log2(groups.abs().amax(2) / E2M1[-1])).clamp(-100, 100)
    size = (groups.abs() * torch.exp2(-exponent)[..., None]).clamp(max=E2M1[-1])
    middles = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device=t.device)
    q = (torch.bucketize(size, middles) + 8 * (groups < 0)).to(torch.uint8).view(rows, -1)[:, :columns + columns % 2]
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), (exponent + 127).to(torch.uint8)


def _logits(tokens, experts, padded, dtype, g):
    """A router's: some experts are liked better than others, and padding likes none."""
    z = torch.randn((tokens, experts), device="cuda", generator=g) * 1.5 + torch.randn(experts, device="cuda", generator=g) * 0.5
    if padded:
        z[torch.rand(tokens, device="cuda", generator=g) < padded] = -math.inf
    return z.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, by=1.0):
        return torch.randn(shape, device="cuda", generator=g) * by

    def stream(rows, columns):
        """Hidden states: one channel in a hundred is eight times as large as the others."""
        return normal(rows, columns) * (1.0 + 7.0 * (torch.rand(columns, device="cuda", generator=g) < 0.01))

    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if kind.startswith("four_bit"):
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = stream(M, K).to(dtype)
        s["weights"], s["weight_scales"] = map(list, zip(*[_rows_in_4_bits(normal(N, K, by=K ** -0.5)) for _ in range(2 if kind == "four_bit_gated" else 1)]))
        if kind == "four_bit":
            s["bias"] = normal(N, by=0.1).to(dtype) if case["bias"] else None
            s["residual"] = stream(M, N).to(dtype) if case["residual"] else None
        return s
    tokens, k = case["tokens"], case["k"]
    if kind.startswith("route"):
        s["logits"] = _logits(tokens, case["experts"], case["padded"], dtype, g)
        if kind == "route_backward":
            s["experts"] = _choose(s["logits"], k)
            s["dweights"] = normal(tokens, k)
        return s
    # what the router left: places by expert, and the tokens in them
    experts = case.get("experts", 16)
    route = _route(_logits(tokens, max(experts, k), case.get("padded", 0.0), torch.float32, g), k, True)
    s["offsets"], s["rows"], s["places"] = route["offsets"], route["rows"], route["places"]
    s["ends"] = s["offsets"].tolist()                           # (only the plain form reads them: a loop over the experts)
    places = tokens * k
    if kind.startswith("combine"):
        N = case["N"]
        s["x"] = normal(places, N).to(dtype)
        s["weights"] = route["weights"] if case.get("weights", True) else None
        if kind == "combine":
            s["residual"] = stream(tokens, N).to(dtype) if case["residual"] else None
        else:
            s["dy"] = normal(tokens, N, by=0.1).to(dtype)
        return s
    N, K = case["N"], case["K"]
    eight, gated, down = case["dtype"] == "float8", "gated" in kind, "linear" in kind
    x = normal(places, K) if down else stream(tokens, K)        # (the down projection's rows are grouped already)
    weights = [normal(experts, N, K, by=K ** -0.5) for _ in range(2 if gated else 1)]
    if eight:
        s["x"], s["x_scale"] = _rows_in_8_bits(x)
        s["weights"], s["weight_scales"] = map(list, zip(*[_rows_in_8_bits(w) for w in weights]))
    else:
        s["x"], s["x_scale"] = x.to(dtype), None
        s["weights"], s["weight_scales"] = [w.to(dtype) for w in weights], [None] * len(weights)
    if down:
        s["rows"] = None
    if kind.endswith("backward"):
        s["dy"] = normal(places, N, by=0.1).to(dtype)
        if gated:
            s["gate"], s["up"] = normal(places, N).to(dtype), normal(places, N).to(dtype)
    return s


# ---------------------------------------------------------------- the framework's operators

def _run_own(s):
    from tiramisu_amd import operators

    c = s["case"]
    kind = c["kind"]
    if kind == "route":
        r = operators.route(s["logits"], c["k"], normalise=c["normalise"])
        return {"experts": r.experts, "weights": r.weights, "offsets": r.offsets, "rows": r.rows, "places": r.places}
    if kind == "route_backward":
        return {"dlogits": operators.route_backward(s["dweights"], s["logits"], s["experts"], normalise=c["normalise"])}
    if kind == "grouped_linear":
        return {"y": operators.grouped_linear(s["x"], s["weights"][0], s["offsets"], x_scale=s["x_scale"], weight_scale=s["weight_scales"][0])}
    if kind == "grouped_linear_backward":
        r = operators.grouped_linear_backward(s["dy"], s["x"], s["weights"][0], s["offsets"])
        return {"dx": r.dx, "dweight": r.dweight}
    if kind == "grouped_gated":
        r = operators.grouped_gated_linear(s["x"], s["weights"][0], s["weights"][1], s["offsets"], rows=s["rows"], activation=c["activation"], x_scale=s["x_scale"],
                                           gate_scale=s["weight_scales"][0], up_scale=s["weight_scales"][1], keep_pre=c["keep"])
        return {"h": r.h, "gate": r.gate, "up": r.up}
    if kind == "grouped_gated_backward":
        r = operators.grouped_gated_linear_backward(s["dy"], s["x"], s["weights"][0], s["weights"][1], s["gate"], s["up"], s["offsets"], rows=s["rows"], activation=c["activation"])
        return {"dx": r.dx, "dgate_weight": r.dgate_weight, "dup_weight": r.dup_weight}
    if kind == "combine":
        return {"y": operators.combine(s["x"], s["places"], weights=s["weights"], residual=s["residual"])}
    if kind == "combine_backward":
        r = operators.combine_backward(s["dy"], s["x"], s["places"], s["weights"], s["rows"])
        return {"dx": r.dx, "dweights": r.dweights}
    if kind == "four_bit":
        r = operators.four_bit_linear(s["x"], s["weights"][0], s["weight_scales"][0], bias=s["bias"], residual=s["residual"], activation=c["activation"])
        return {"y": r.y}
    r = operators.four_bit_gated_linear(s["x"], s["weights"][0], s["weights"][1], s["weight_scales"][0], s["weight_scales"][1], activation=c["activation"])
    return {"h": r.h}


# ---------------------------------------------------------------- the plain forms: 32 bits, rounded once at the end

def _choose(logits, k):
    """The k largest of every row, the lowest index first among equal ones; -1 where minus infinity is all that is left."""
    value, index = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    return torch.where(value[:, :k] == -math.inf, -1, index[:, :k]).to(torch.int32)


def _chosen_weights(logits, experts, normalise):
    """The chosen ones' share of their sum, or of all."""
    z = logits.float()
    there = experts >= 0
    most = torch.where(there[:, :1], z.amax(1, keepdim=True), 0.0)
    chosen = torch.where(there, torch.exp(torch.gather(z, 1, experts.clamp(min=0).long()) - most), 0.0)
    total = (chosen if normalise else torch.exp(z - most)).sum(1, keepdim=True)
    return torch.where(there, chosen / total, 0.0)


def _route(logits, k, normalise):
    tokens, count = logits.shape
    experts = _choose(logits, k)
    flat = torch.where(experts < 0, count, experts).view(-1)
    ordered, order = torch.sort(flat, stable=True)
    there = ordered < count
    rows = torch.where(there, order // k, -1).to(torch.int32)
    offsets = torch.searchsorted(ordered, torch.arange(count + 1, device=logits.device, dtype=torch.int32), out_int32=True)
    places = torch.empty_like(flat)
    places[order] = torch.where(there, torch.arange(len(flat), device=logits.device), -1).to(torch.int32)
    return {"experts": experts, "weights": _chosen_weights(logits, experts, normalise), "offsets": offsets, "rows": rows, "places": places.view(tokens, k)}


def _activation(name, z):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def _activation_slope(name, z):
    if name == "relu":
        return (z > 0).float()
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * z * z)
    p = torch.sigmoid(z)
    return p * (1.0 + z * (1.0 - p))


def _widened(q, scale, columns):
    """4-bit rows as the numbers that they stand for."""
    codes = torch.stack((q & 15, q >> 4), 2).view(q.shape[0], -1)[:, :columns].long()
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)[codes]
    return value * torch.exp2(scale.float() - 127.0).repeat_interleave(GROUP, 1)[:, :columns]


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "route":
        return _route(s["logits"], c["k"], c["normalise"])
    if kind == "route_backward":
        w = _chosen_weights(s["logits"], s["experts"], c["normalise"])
        there = s["experts"] >= 0
        dot = (w * s["dweights"]).sum(1, keepdim=True)
        index = torch.where(there, s["experts"], c["experts"]).long()
        if c["normalise"]:
            dz = torch.zeros((c["tokens"], c["experts"] + 1), device="cuda")
            dz.scatter_(1, index, w * (s["dweights"] - dot))
        else:
            z = s["logits"].float()
            p = torch.where(there[:, :1], torch.exp(z - torch.where(there[:, :1], z.amax(1, keepdim=True), 0.0)), 0.0)
            p = p / torch.where(there[:, :1], p.sum(1, keepdim=True), 1.0)
            dz = torch.nn.functional.pad(-p * dot, (0, 1))
            dz.scatter_add_(1, index, w * s["dweights"])
        return {"dlogits": dz[:, :-1].to(s["logits"].dtype)}
    half = torch.bfloat16 if c["dtype"] == "float8" else DTYPES[c["dtype"]]
    if kind.startswith("four_bit"):
        x = s["x"].float()
        z = [x @ _widened(q, v, c["K"]).t() for q, v in zip(s["weights"], s["weight_scales"])]
        if kind == "four_bit_gated":
            return {"h": (_activation(c["activation"], z[0]) * z[1]).to(half)}
        y = _activation(c["activation"], z[0] + s["bias"].float() if c["bias"] else z[0])
        return {"y": (y + s["residual"].float() if c["residual"] else y).to(half)}
    if kind.startswith("combine"):
        there = s["places"] >= 0
        gathered = torch.where(there[..., None], s["x"].float()[s["places"].clamp(min=0).long()], 0.0)
        if kind == "combine":
            y = (gathered * s["weights"][..., None]).sum(1) if c["weights"] else gathered.sum(1)
            return {"y": (y + s["residual"].float() if c["residual"] else y).to(half)}
        dy = s["dy"].float()
        dx = torch.zeros((len(s["x"]) + 1, c["N"]), device="cuda")
        dx[torch.where(there, s["places"], len(s["x"])).long().view(-1)] = (s["weights"][..., None] * dy[:, None]).view(-1, c["N"])
        return {"dx": dx[:-1].to(half), "dweights": (gathered * dy[:, None]).sum(2)}
    # the products, expert by expert
    x = s["x"].float() if s["rows"] is None else s["x"].float()[s["rows"].clamp(min=0).long()]
    if s["x_scale"] is not None:
        x = x * (s["x_scale"] if s["rows"] is None else s["x_scale"][s["rows"].clamp(min=0).long()])[:, None]
    ends = s["ends"]
    groups = [(e, slice(ends[e], ends[e + 1])) for e in range(c["experts"]) if ends[e + 1] > ends[e]]

    def weight(i, e):
        w = s["weights"][i][e].float()
        return w if s["weight_scales"][i] is None else w * s["weight_scales"][i][e][:, None]

    def of_rows(columns):
        return torch.zeros((c["tokens"] * c["k"], columns), device="cuda")

    if not kind.endswith("backward"):
        z = [of_rows(c["N"]) for _ in s["weights"]]
        for e, at in groups:
            for i, out in enumerate(z):
                out[at] = x[at] @ weight(i, e).t()
        if kind == "grouped_linear":
            return {"y": z[0].to(half)}
        return {"h": (_activation(c["activation"], z[0]) * z[1]).to(half), "gate": z[0].to(half) if c["keep"] else None, "up": z[1].to(half) if c["keep"] else None}
    dy = s["dy"].float()
    if kind == "grouped_linear_backward":
        dz = [dy]
    else:
        gate = s["gate"].float()
        dz = [dy * s["up"].float() * _activation_slope(c["activation"], gate), dy * _activation(c["activation"], gate)]
    dx, dweights = of_rows(c["K"]), [torch.zeros((c["experts"], c["N"], c["K"]), device="cuda") for _ in dz]
    for e, at in groups:
        for i, d in enumerate(dz):
            dx[at] += d[at] @ weight(i, e)
            dweights[i][e] = d[at].t() @ x[at]
    if kind == "grouped_linear_backward":
        return {"dx": dx.to(half), "dweight": dweights[0].to(half)}
    return {"dx": dx.to(half), "dgate_weight": dweights[0].to(half), "dup_weight": dweights[1].to(half)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind, e = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind.startswith("four_bit"):
        M, N, K = case["M"], case["N"], case["K"]
        w = 2 if kind == "four_bit_gated" else 1
        weights = w * N * ((K + 1) // 2 + (K + GROUP - 1) // GROUP)
        return {"bytes": weights + 2 * M * K + 2 * M * N * (1 + case.get("residual", False)) + 2 * N * case.get("bias", False), "flops": 2 * w * M * N * K}
    T, k = case["tokens"], case["k"]
    S = T * k
    if kind == "route":
        return {"bytes": T * case["experts"] * e + 16 * S + 4 * (case["experts"] + 1), "flops": 4 * T * case["experts"]}
    if kind == "route_backward":
        return {"bytes": 2 * T * case["experts"] * e + 8 * S, "flops": 4 * T * case["experts"]}
    if kind == "combine":
        return {"bytes": 2 * case["N"] * (S + T * (1 + case["residual"])) + 4 * S * (1 + case["weights"]), "flops": 2 * S * case["N"]}
    if kind == "combine_backward":
        return {"bytes": 2 * case["N"] * (2 * S + T) + 16 * S, "flops": 3 * S * case["N"]}
    E, N, K = case["experts"], case["N"], case["K"]
    w = 2 if "gated" in kind else 1
    chosen = E * (1.0 - (1.0 - k / E) ** T)                    # experts that some token chose, were they all liked alike
    rows = S if "linear" in kind else T
    b = rows * K * e + int(chosen * w * N * K * e)
    if kind.endswith("backward"):
        b += 2 * (S * K + w * E * N * K) + 2 * S * N * (3 if w == 2 else 1)
        return {"bytes": b, "flops": 4 * w * S * N * K}
    b += 2 * S * N * (3 if case.get("keep") else 1)
    if e == 1:
        b += 4 * rows + int(4 * chosen * w * N)
    return {"bytes": b + 4 * (E + 1) + (4 * S if w == 2 else 0), "flops": 2 * w * S * N * K}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_activation(name, z):
    """Written with other functions than the plain form's, and differentiable: gradients are autograd's."""
    if name == "relu":
        return 0.5 * (z + z.abs())
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z.pow(3))))
    if name == "silu":
        return 0.5 * z * (1.0 + torch.tanh(0.5 * z))
    return z


def _exact_route(logits, k, normalise):
    """One choice after the other; places by counting."""
    z = logits.double()
    tokens, count = z.shape
    left, number = z.clone(), torch.arange(count, device=z.device)
    experts = []
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        first = torch.where(left == best, number, count).min(1).values
        experts.append(torch.where(best[:, 0] == -math.inf, -1, first))
        left.scatter_(1, first[:, None], -math.inf)
    experts = torch.stack(experts, 1)
    taken = (experts[..., None] == number).any(1)
    p = torch.softmax(torch.where(taken, z, -math.inf) if normalise else z, 1)
    weights = torch.where(experts >= 0, torch.gather(p, 1, experts.clamp(min=0)), 0.0)
    places = torch.full((tokens * k,), -1, device=z.device, dtype=torch.int64)
    rows, offsets, flat = torch.full_like(places, -1), [0], experts.view(-1)
    for e in range(count):
        at = torch.nonzero(flat == e)[:, 0]
        places[at] = offsets[-1] + torch.arange(len(at), device=z.device)
        rows[offsets[-1]:offsets[-1] + len(at)] = at // k
        offsets.append(offsets[-1] + len(at))
    whole = {"experts": experts, "offsets": torch.tensor(offsets, device=z.device), "rows": rows, "places": places.view(tokens, k)}
    return dict({name: t.to(torch.int32) for name, t in whole.items()}, weights=weights)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def wide(t):
        return None if t is None else t.double()

    if kind == "route":
        r = _exact_route(s["logits"], case["k"], case["normalise"])
        return {name: r[name] for name in ("experts", "weights", "offsets", "rows", "places")}
    if kind == "route_backward":
        # autograd through the chosen ones' softmax; rows without an expert have no gradient
        alive = s["experts"][:, 0] >= 0
        z = wide(s["logits"][alive]).requires_grad_()
        experts = s["experts"][alive]
        taken = torch.zeros(z.shape, dtype=torch.bool, device=z.device).scatter_(1, experts.clamp(min=0).long(), True)
        p = torch.softmax(z.masked_fill(~taken, -math.inf) if case["normalise"] else z, 1)
        there = experts >= 0
        w = torch.where(there, torch.gather(p, 1, experts.clamp(min=0).long()), 0.0)
        out = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
        out[alive] = torch.autograd.grad(w, z, wide(s["dweights"][alive]))[0]
        return {"dlogits": out}
    if kind.startswith("four_bit"):
        K = case["K"]
        weights = []
        for q, scale in zip(s["weights"], s["weight_scales"]):
            code = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.int64, device="cuda")
            code[:, 0::2], code[:, 1::2] = (q & 15).long(), (q >> 4).long()
            code = code[:, :K]
            # sign, two bits of exponent (bias 1), one of mantissa
            exponent, mantissa = (code >> 1) & 3, (code & 1).double()
            value = torch.where(exponent > 0, (1.0 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1.0), 0.5 * mantissa) * (1.0 - 2.0 * (code >> 3).double())
            weights.append(torch.ldexp(value, scale.long()[:, torch.arange(K, device="cuda") // GROUP] - 127))
        z = [torch.mm(wide(s["x"]), w.t().contiguous()) for w in weights]
        if kind == "four_bit_gated":
            return {"h": z[1] * _exact_activation(case["activation"], z[0])}
        y = _exact_activation(case["activation"], z[0] + wide(s["bias"]) if case["bias"] else z[0])
        return {"y": y + wide(s["residual"]) if case["residual"] else y}
    if kind == "combine":
        y = torch.zeros((case["tokens"], case["N"]), dtype=torch.float64, device="cuda") if s["residual"] is None else wide(s["residual"])
        x = wide(s["x"])
        for j in range(case["k"]):
            at = s["places"][:, j]
            factor = (at >= 0).double() if s["weights"] is None else torch.where(at >= 0, wide(s["weights"][:, j]), 0.0)
            y = y + factor[:, None] * x[at.clamp(min=0).long()]
        return {"y": y}
    if kind == "combine_backward":
        x, dy = wide(s["x"]), wide(s["dy"])
        dx, dweights = torch.zeros_like(x), torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            t = torch.nonzero(s["places"][:, j] >= 0)[:, 0]
            at = s["places"][t, j].long()
            dx[at] = wide(s["weights"][t, j])[:, None] * dy[t]
            dweights[t, j] = torch.linalg.vecdot(dy[t], x[at])
        return {"dx": dx, "dweights": dweights}
    ends = s["offsets"].tolist()
    x = wide(s["x"]) if s["x_scale"] is None else wide(s["x"]) * wide(s["x_scale"])[:, None]
    if s["rows"] is not None:
        x = torch.cat([x[s["rows"][:ends[-1]].long()], torch.zeros((len(s["rows"]) - ends[-1], case["K"]), dtype=torch.float64, device="cuda")])
    count, backward = len(s["weights"]), kind.endswith("backward")
    if backward:
        dz = [wide(s["dy"])]
        if count == 2:
            gate, up = wide(s["gate"]).requires_grad_(), wide(s["up"]).requires_grad_()
            dz = torch.autograd.grad(_exact_activation(case["activation"], gate) * up, (gate, up), dz[0])
        dx, dweights = torch.zeros_like(x), [torch.zeros(w.shape, dtype=torch.float64, device="cuda") for w in s["weights"]]
    else:
        z = [torch.zeros((len(x), case["N"]), dtype=torch.float64, device="cuda") for _ in s["weights"]]
    for e in range(case["experts"]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        for i in range(count):
            w = wide(s["weights"][i][e])
            if s["weight_scales"][i] is not None:
                w = w * wide(s["weight_scales"][i][e])[:, None]
            if backward:
                dx[a:b] += torch.mm(dz[i][a:b], w)
                dweights[i][e] = torch.mm(dz[i][a:b].t().contiguous(), x[a:b])
            else:
                z[i][a:b] = torch.mm(x[a:b], w.t().contiguous())
    if backward:
        return {"dx": dx, "dweight": dweights[0]} if count == 1 else {"dx": dx, "dgate_weight": dweights[0], "dup_weight": dweights[1]}
    if count == 1:
        return {"y": z[0]}
    return {"h": z[1] * _exact_activation(case["activation"], z[0]), "gate": z[0] if case["keep"] else None, "up": z[1] if case["keep"] else None}
