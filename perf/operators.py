"""The operators of a transformer's feed-forward sublayer, as a program of their user runs them.

Three operators, each forward and backward, and from one token to a long prompt or a training batch:

* norm:   the residual stream's addition, the root-mean-square norm of the sum, its result in 16 or 32 bits or in 8 bits
          (e4m3, with one scale for each row);
* linear: a matrix product with bias, activation and residual in its epilogue, on 16-bit operands or on 8-bit ones with scales;
* gated:  both projections of a gated feed-forward layer, the activation of the one and the product with the other.

Weights are [outputs, inputs], rows of x are tokens.  All tensors live on the GPU.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32, "float8": torch.float8_e4m3fn}
EPS = 1e-6
E4M3_MOST = 448.0


def listed():
    return [
        # serving, one token: the norm ahead of an 8-bit product, where a launch is all that it costs
        {"name": "norm one token to 8 bits", "kind": "norm", "rows": 1, "columns": 4096, "dtype": "bfloat16", "residual": True, "eight_bit": True, "keep": False},
        # training at a size that nothing divides, keeping what the backward pass reads
        {"name": "norm ragged, kept", "kind": "norm", "rows": 2000, "columns": 1430, "dtype": "float16", "residual": True, "eight_bit": False, "keep": True},
        # a long prompt through the residual stream
        {"name": "norm long prompt", "kind": "norm", "rows": 16384, "columns": 4096, "dtype": "bfloat16", "residual": True, "eight_bit": False, "keep": False},
        # training: a batch's backward pass, with the gradient that arrives along the residual stream
        {"name": "norm backward", "kind": "norm_backward", "rows": 8192, "columns": 2048, "dtype": "bfloat16", "residual": True},
        # serving, one token: the output projection with bias and residual, bound by the weights' bytes
        {"name": "linear one token", "kind": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bfloat16", "activation": "none", "bias": True, "residual": True, "keep": False},
        # training at a size that no tile divides, keeping the sums ahead of the activation
        {"name": "linear ragged, kept", "kind": "linear", "M": 2000, "N": 1500, "K": 1000, "dtype": "float16", "activation": "gelu", "bias": True, "residual": False, "keep": True},
        # a prompt through the down projection in 8 bits, added to the residual stream
        {"name": "linear 8 bits", "kind": "linear", "M": 4096, "N": 4096, "K": 4096, "dtype": "float8", "activation": "none", "bias": False, "residual": True, "keep": False},
        # training: gradients of input, weights and bias through the activation
        {"name": "linear backward", "kind": "linear_backward", "M": 4096, "N": 4096, "K": 1024, "dtype": "bfloat16", "activation": "gelu", "bias": True},
        # serving, sixteen sequences by a token each
        {"name": "gated 16 tokens", "kind": "gated", "M": 16, "N": 8192, "K": 2048, "dtype": "bfloat16", "activation": "silu", "keep": False},
        # a long prompt, or a training batch, through a wide layer
        {"name": "gated prompt", "kind": "gated", "M": 4096, "N": 8192, "K": 4096, "dtype": "bfloat16", "activation": "silu", "keep": True},
        # a ragged batch in 8 bits
        {"name": "gated ragged 8 bits", "kind": "gated", "M": 1000, "N": 1500, "K": 700, "dtype": "float8", "activation": "silu", "keep": False},
        # training: gradients of input and both weights
        {"name": "gated backward", "kind": "gated_backward", "M": 4096, "N": 4096, "K": 2048, "dtype": "bfloat16", "activation": "silu"},
    ]


def draw(rng):
    def size(low, high, step=1):
        """Spread over the logarithm; half of the sizes are what they are, half a multiple of `step`."""
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        if step > 1 and rng.random() < 0.5:
            v = (v + step // 2) // step * step
        return max(low, min(high, v))

    kind = rng.choice(["norm", "norm_backward", "linear", "linear_backward", "gated", "gated_backward"])
    if kind == "norm":
        eight_bit = rng.random() < 0.4
        return {"kind": kind, "rows": size(1, 16384), "columns": size(64, 4096, 64), "dtype": rng.choice(["bfloat16", "float16", "float32"]),
                "residual": rng.random() < 0.7, "eight_bit": eight_bit, "keep": not eight_bit and rng.random() < 0.5}
    if kind == "norm_backward":
        return {"kind": kind, "rows": size(64, 8192), "columns": size(64, 4096, 64), "dtype": rng.choice(["bfloat16", "float16", "float32"]), "residual": rng.random() < 0.7}
    if kind == "linear":
        dtype = rng.choice(["bfloat16", "float16", "float8"])
        activation = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        return {"kind": kind, "M": size(1, 4096, 16), "N": size(64, 4096, 64), "K": size(64, 4096, 64), "dtype": dtype, "activation": activation,
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "keep": activation != "none" and rng.random() < 0.5}
    if kind == "linear_backward":
        return {"kind": kind, "M": size(64, 4096, 16), "N": size(64, 4096, 64), "K": size(64, 2048, 64), "dtype": rng.choice(["bfloat16", "float16"]),
                "activation": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.5}
    if kind == "gated":
        dtype = rng.choice(["bfloat16", "float16", "float8"])
        return {"kind": kind, "M": size(1, 4096, 16), "N": size(64, 8192, 64), "K": size(64, 4096, 64), "dtype": dtype,
                "activation": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), "keep": rng.random() < 0.4}
    return {"kind": kind, "M": size(64, 4096, 16), "N": size(64, 4096, 64), "K": size(64, 2048, 64), "dtype": rng.choice(["bfloat16", "float16"]),
            "activation": rng.choice(["silu", "gelu", "gelu_tanh", "relu"])}


# ---------------------------------------------------------------- inputs

def _rows_in_8_bits(t):
    """What a program that serves in 8 bits keeps of a matrix: e4m3 values and one scale for each row."""
    scale = t.abs().amax(1) / E4M3_MOST
    return (t / scale[:, None]).to(torch.float8_e4m3fn), scale


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
    if kind in ("norm", "norm_backward"):
        rows, columns = case["rows"], case["columns"]
        s["weight"] = (1.0 + normal(columns, by=0.1)).to(dtype)
        x = stream(rows, columns)
        if kind == "norm":
            s["x"] = x.to(dtype)
            s["residual"] = stream(rows, columns).to(dtype) if case["residual"] else None
        else:
            s["sum"] = x.to(dtype)
            s["rstd"] = torch.rsqrt(s["sum"].float().square().mean(1) + EPS)
            s["dy"] = normal(rows, columns, by=0.1).to(dtype)
            s["dsum"] = normal(rows, columns, by=0.1).to(dtype) if case["residual"] else None
        return s
    M, N, K = case["M"], case["N"], case["K"]
    eight = case["dtype"] == "float8"
    x = stream(M, K)
    weights = [normal(N, K, by=K ** -0.5) for _ in range(2 if kind.startswith("gated") else 1)]
    if eight:
        s["x"], s["x_scale"] = _rows_in_8_bits(x)
        s["weights"], s["weight_scales"] = map(list, zip(*[_rows_in_8_bits(w) for w in weights]))
    else:
        s["x"], s["x_scale"] = x.to(dtype), None
        s["weights"], s["weight_scales"] = [w.to(dtype) for w in weights], [None] * len(weights)
    half = torch.bfloat16 if eight else dtype
    if kind == "linear":
        s["bias"] = normal(N, by=0.1).to(half) if case["bias"] else None
        s["residual"] = stream(M, N).to(half) if case["residual"] else None
    elif kind == "linear_backward":
        s["dy"] = normal(M, N, by=0.1).to(half)
        s["pre"] = (s["x"].float() @ s["weights"][0].float().t()).to(half) if case["activation"] != "none" else None
    elif kind == "gated_backward":
        s["dh"] = normal(M, N, by=0.1).to(half)
        s["gate"], s["up"] = [(s["x"].float() @ w.float().t()).to(half) for w in s["weights"]]
    return s


# ---------------------------------------------------------------- the framework's operators

def _run_own(s):
    from tiramisu_amd import operators

    c = s["case"]
    kind = c["kind"]
    if kind == "norm":
        r = operators.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, eight_bit=c["eight_bit"], keep_rstd=c["keep"])
        return {"y": r.y, "sum": r.sum if c["residual"] else None, "scale": r.scale, "rstd": r.rstd}
    if kind == "norm_backward":
        r = operators.rms_norm_backward(s["dy"], s["sum"], s["weight"], s["rstd"], dsum=s["dsum"])
        return {"dx": r.dx, "dweight": r.dweight}
    if kind == "linear":
        r = operators.linear(s["x"], s["weights"][0], bias=s["bias"], residual=s["residual"], activation=c["activation"],
                             x_scale=s["x_scale"], weight_scale=s["weight_scales"][0], keep_pre=c["keep"])
        return {"y": r.y, "pre": r.pre}
    if kind == "linear_backward":
        r = operators.linear_backward(s["dy"], s["x"], s["weights"][0], pre=s["pre"], activation=c["activation"], bias=c["bias"])
        return {"dx": r.dx, "dweight": r.dweight, "dbias": r.dbias}
    if kind == "gated":
        r = operators.gated_linear(s["x"], s["weights"][0], s["weights"][1], activation=c["activation"], x_scale=s["x_scale"],
                                   gate_scale=s["weight_scales"][0], up_scale=s["weight_scales"][1], keep_pre=c["keep"])
        return {"h": r.h, "gate": r.gate, "up": r.up}
    r = operators.gated_linear_backward(s["dh"], s["x"], s["weights"][0], s["weights"][1], s["gate"], s["up"], activation=c["activation"])
    return {"dx": r.dx, "dgate_weight": r.dgate_weight, "dup_weight": r.dup_weight}


# ---------------------------------------------------------------- the plain forms: 32 bits, rounded once at the end

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
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1.0 + z * (1.0 - p))
    return torch.ones_like(z)


def _product(x, x_scale, weight, weight_scale):
    z = x.float() @ weight.float().t()
    return z if x_scale is None else z * x_scale[:, None] * weight_scale


def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "norm":
        x, dtype = s["x"].float(), s["x"].dtype
        if c["residual"]:
            x = x + s["residual"].float()
        rstd = torch.rsqrt((x * x).mean(1) + EPS)
        y = x * rstd[:, None] * s["weight"].float()
        scale = None
        if c["eight_bit"]:
            scale = y.abs().amax(1) / E4M3_MOST
            y = (y / scale[:, None]).to(torch.float8_e4m3fn)
        else:
            y = y.to(dtype)
        return {"y": y, "sum": x.to(dtype) if c["residual"] else None, "scale": scale, "rstd": rstd if c["keep"] else None}
    if kind == "norm_backward":
        dtype = s["sum"].dtype
        xhat = s["sum"].float() * s["rstd"][:, None]
        dy = s["dy"].float()
        dxhat = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (dxhat - xhat * (dxhat * xhat).mean(1, keepdim=True))
        if c["residual"]:
            dx = dx + s["dsum"].float()
        return {"dx": dx.to(dtype), "dweight": (dy * xhat).sum(0).to(dtype)}
    half = torch.bfloat16 if c["dtype"] == "float8" else s["x"].dtype
    if kind == "linear":
        z = _product(s["x"], s["x_scale"], s["weights"][0], s["weight_scales"][0])
        if c["bias"]:
            z = z + s["bias"].float()
        y = _activation(c["activation"], z)
        if c["residual"]:
            y = y + s["residual"].float()
        return {"y": y.to(half), "pre": z.to(half) if c["keep"] else None}
    if kind == "linear_backward":
        dz = s["dy"].float()
        if c["activation"] != "none":
            dz = dz * _activation_slope(c["activation"], s["pre"].float())
        return {"dx": (dz @ s["weights"][0].float()).to(half), "dweight": (dz.t() @ s["x"].float()).to(half), "dbias": dz.sum(0).to(half) if c["bias"] else None}
    if kind == "gated":
        gate, up = [_product(s["x"], s["x_scale"], w, v) for w, v in zip(s["weights"], s["weight_scales"])]
        h = _activation(c["activation"], gate) * up
        return {"h": h.to(half), "gate": gate.to(half) if c["keep"] else None, "up": up.to(half) if c["keep"] else None}
    dh, gate, up, x = s["dh"].float(), s["gate"].float(), s["up"].float(), s["x"].float()
    dgate = dh * up * _activation_slope(c["activation"], gate)
    dup = dh * _activation(c["activation"], gate)
    return {"dx": (dgate @ s["weights"][0].float() + dup @ s["weights"][1].float()).to(half),
            "dgate_weight": (dgate.t() @ x).to(half), "dup_weight": (dup.t() @ x).to(half)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        e, n, columns = DTYPES[case["dtype"]].itemsize, case["rows"] * case["columns"], case["columns"]
        if kind == "norm":
            b = n * e * (3 if case["residual"] else 1) + columns * e                       # x, residual and sum; the weight
            b += n + 4 * case["rows"] if case["eight_bit"] else n * e                       # y
            return {"bytes": b + (4 * case["rows"] if case["keep"] else 0), "flops": 6 * n}
        return {"bytes": n * e * (4 if case["residual"] else 3) + 2 * columns * e + 4 * case["rows"], "flops": 12 * n}
    M, N, K = case["M"], case["N"], case["K"]
    e = DTYPES[case["dtype"]].itemsize
    w = 2 if kind.startswith("gated") else 1                                                # weights
    b = (M * K + w * N * K) * e
    if kind == "linear":
        b += 2 * (M * N * (1 + case["residual"] + case["keep"]) + N * case["bias"]) + (4 * (M + N) if e == 1 else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    if kind == "gated":
        b += 2 * M * N * (3 if case["keep"] else 1) + (4 * (M + 2 * N) if e == 1 else 0)
        return {"bytes": b, "flops": 4 * M * N * K}
    b += 2 * (M * K + w * N * K)                                                            # dx and the weights' gradients
    if kind == "linear_backward":
        return {"bytes": b + 2 * (M * N * (1 + (case["activation"] != "none")) + N * case["bias"]), "flops": 4 * M * N * K}
    return {"bytes": b + 2 * 3 * M * N, "flops": 8 * M * N * K}


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


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def wide(t):
        return None if t is None else t.double()

    if kind == "norm":
        x = wide(s["x"]) if not case["residual"] else wide(s["x"]) + wide(s["residual"])
        length = torch.sqrt(torch.linalg.vector_norm(x, dim=1).square() / case["columns"] + EPS)
        y = x / length[:, None] * wide(s["weight"])
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / E4M3_MOST if case["eight_bit"] else None
        # in 8 bits: the numbers that the 8-bit values stand for, ahead of their rounding
        return {"y": y if scale is None else y / scale[:, None], "sum": x if case["residual"] else None, "scale": scale,
                "rstd": 1.0 / length if case["keep"] else None}
    if kind == "norm_backward":
        # sum / length(sum) in general; here 1 / length is given, and the gradient of length follows from it
        x, dy, w, rstd = wide(s["sum"]), wide(s["dy"]), wide(s["weight"]), wide(s["rstd"])[:, None]
        dot = torch.sum(dy * w * x, 1, keepdim=True) / case["columns"]
        dx = dy * w * rstd - dot * x * rstd.pow(3)
        return {"dx": dx if s["dsum"] is None else dx + wide(s["dsum"]), "dweight": torch.sum(dy * (x * rstd), 0)}
    x = wide(s["x"]) if s["x_scale"] is None else wide(s["x"]) * wide(s["x_scale"])[:, None]
    weights = [wide(w) if v is None else wide(w) * wide(v)[:, None] for w, v in zip(s["weights"], s["weight_scales"])]
    if kind == "linear":
        z = torch.mm(x, weights[0].t().contiguous())
        if case["bias"]:
            z = z + wide(s["bias"])
        y = _exact_activation(case["activation"], z)
        return {"y": y + wide(s["residual"]) if case["residual"] else y, "pre": z if case["keep"] else None}
    if kind == "gated":
        gate, up = [torch.mm(x, w.t().contiguous()) for w in weights]
        return {"h": up * _exact_activation(case["activation"], gate), "gate": gate if case["keep"] else None, "up": up if case["keep"] else None}
    if kind == "linear_backward":
        dz = wide(s["dy"])
        if case["activation"] != "none":
            z = wide(s["pre"]).requires_grad_()
            dz, = torch.autograd.grad(_exact_activation(case["activation"], z), z, dz)
        return {"dx": torch.mm(dz, weights[0]), "dweight": torch.mm(dz.t().contiguous(), x), "dbias": dz.sum(0) if case["bias"] else None}
    gate, up = wide(s["gate"]).requires_grad_(), wide(s["up"]).requires_grad_()
    dgate, dup = torch.autograd.grad(_exact_activation(case["activation"], gate) * up, (gate, up), wide(s["dh"]))
    return {"dx": torch.mm(dgate, weights[0]) + torch.mm(dup, weights[1]),
            "dgate_weight": torch.mm(dgate.t().contiguous(), x), "dup_weight": torch.mm(dup.t().contiguous(), x)}
