"""The operators of a transformer's feed-forward sublayer on torch tensors: the residual stream's addition and root-mean-square norm, the matrix
product with bias, activation and residual in its epilogue, and both projections of a gated feed-forward layer in one
kernel; each with its backward pass, on 16-bit operands or (forward) 8-bit ones with scales.

These functions check their arguments, allocate the results and call the runtime's C ABI (include/tiramisu_hip_wrappers.h), whose
kernels run on torch's current stream of the tensors' device; nothing waits for them.  Leading dimensions are tokens: x of shape
[..., K] gives a result of shape [..., N].  Weights are [outputs, inputs].  Tensors need dense rows (stride 1 in the last
dimension), with one stride from row to row; others are refused, never copied silently.  Results are new, dense tensors.
ValueError says what does not fit, RuntimeError that the runtime refused the call (its reason is on stderr).
"""
import struct
from typing import NamedTuple, Optional

import torch

from . import runtime

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
_HALVES = (torch.float16, torch.bfloat16)
_NORM_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_PRODUCT_TYPES = _HALVES + (torch.float8_e4m3fn,)

# The operators of the C ABI: number, and how their arguments are packed for tiramisu_hip_operator (a call of 16 converted arguments and three for the
# stream cost 2 us more; a norm of one token 12.9 us a call then, of which 5 are the kernel)
_RMS_NORM = 0, struct.Struct("=11Qf4x2Q").pack
_RMS_NORM_BACKWARD = 1, struct.Struct("=13Q").pack
_QUANTIZE_ROWS = 2, struct.Struct("=7Q").pack
_LINEAR = 3, struct.Struct("=17Q").pack
_LINEAR_BACKWARD = 4, struct.Struct("=16Q").pack
_GATED_LINEAR = 5, struct.Struct("=18Q").pack
_GATED_LINEAR_BACKWARD = 6, struct.Struct("=20Q").pack

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_entry = None                     # tiramisu_hip_operator, from the first call on


class RmsNorm(NamedTuple):
    y: torch.Tensor
    sum: torch.Tensor                       # x + residual; x itself without a residual
    scale: Optional[torch.Tensor] = None    # of each row, where y is in 8 bits
    rstd: Optional[torch.Tensor] = None     # 1 / length of each row, where kept


class RmsNormGradients(NamedTuple):
    dx: torch.Tensor                        # of x and of the residual alike
    dweight: torch.Tensor


class EightBitRows(NamedTuple):
    q: torch.Tensor
    scale: torch.Tensor


class Linear(NamedTuple):
    y: torch.Tensor
    pre: Optional[torch.Tensor] = None      # the sums ahead of the activation, where kept


class LinearGradients(NamedTuple):
    dx: torch.Tensor
    dweight: torch.Tensor
    dbias: Optional[torch.Tensor] = None


class GatedLinear(NamedTuple):
    h: torch.Tensor
    gate: Optional[torch.Tensor] = None     # both projections, where kept
    up: Optional[torch.Tensor] = None


class GatedLinearGradients(NamedTuple):
    dx: torch.Tensor
    dgate_weight: torch.Tensor
    dup_weight: torch.Tensor


# ---------------------------------------------------------------- checks

def _rows(t, name, shape=None, dtypes=()):
    """(rows, elements from row to row) of a tensor on the GPU whose rows are dense."""
    if not isinstance(t, torch.Tensor):
        raise ValueError("%s is a tensor, not %s" % (name, type(t).__name__))
    if t.dtype not in dtypes:
        raise ValueError("%s holds %s: %s are taken here" % (name, t.dtype, ", ".join(str(d) for d in dtypes)))
    if t.dim() < 1:
        raise ValueError("%s has no rows" % name)
    if shape is not None and t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, list(t.shape), list(shape)))
    width = t.shape[-1]
    if not t.is_cuda:
        raise ValueError("%s lives on %s: operators run on the GPU" % (name, t.device))
    rows = t.numel() // width if width else 0
    if t.is_contiguous():
        return rows, width
    if t.stride(-1) != 1 and width > 1:
        raise ValueError("%s: the elements of a row are not next to each other" % name)
    # one stride from row to row: dimensions of one row do not count, the others follow each other
    step, expected = None, None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != expected:
            raise ValueError("%s: rows are not one stride apart" % name)
        expected = stride * size
    if step is None:
        step = width
    if step < width:
        raise ValueError("%s: rows overlap" % name)
    return rows, step


def _matrix(t, name, rows, columns, dtype):
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or (rows is not None and t.shape[0] != rows) or t.shape[1] != columns:
        raise ValueError("%s is a matrix of [%s, %d], not %s" % (name, "outputs" if rows is None else rows, columns, list(t.shape) if isinstance(t, torch.Tensor) else t))
    return _rows(t, name, dtypes=(dtype,))[1]


def _vector(t, name, size, dtype, where):
    """Its address; dense."""
    if not isinstance(t, torch.Tensor) or t.shape != (size,) or t.dtype != dtype or not t.is_cuda or (size > 1 and t.stride(0) != 1):
        raise ValueError("%s is a dense vector of %d %s on the GPU, not %s" % (name, size, dtype, "%s of %s" % (t.dtype, list(t.shape)) if isinstance(t, torch.Tensor) else t))
    return _pointer(t, name, where)


def _pointer(t, name, where):
    if t.get_device() != where:
        raise ValueError("%s lives on another GPU" % name)
    return t.data_ptr()


def _row_scale(t, name, x, rows, where):
    """x_scale: a scale for each row of x, in the shape of its leading dimensions or flat."""
    if isinstance(t, torch.Tensor) and t.shape == x.shape[:-1] and t.is_contiguous():
        t = t.reshape(-1)
    return _vector(t, name, rows, torch.float32, where)


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation %r: one of %s" % (name, ", ".join(ACTIVATIONS)))
    return ACTIVATIONS[name]


def _call(operator, where, *args):
    """One operator of the C ABI on torch's current stream of GPU `where`."""
    global _entry
    if _entry is None:
        _entry = runtime.wrappers().tiramisu_hip_operator
    number, pack = operator
    if where != _device():
        with torch.cuda.device(where):
            return _call(operator, where, *args)
    stream = _raw_stream(where) if _raw_stream else torch.cuda.current_stream(where).cuda_stream
    if _entry(number, pack(*args), stream) != 0:
        raise RuntimeError("the runtime refused the call")


def _like(t, dtype):
    """A new dense tensor of t's shape.  (The fewer arguments, the faster: 0.9 us as it is, 1.1 with both.)"""
    if dtype is t.dtype and t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _new(t, shape, dtype):
    """A new dense tensor on t's GPU."""
    return t.new_empty(shape) if dtype is t.dtype else t.new_empty(shape, dtype=dtype)


_float = {}                       # a tensor of 32-bit numbers on each GPU, for its new_empty (0.9 us; of another type than the tensor's 1.5)


def _row_numbers(t, where):
    """A new 32-bit number for each row of t."""
    f = _float.get(where)
    if f is None:
        f = _float[where] = t.new_empty(1, dtype=torch.float32)
    return f.new_empty(t.shape[:-1])


def _eight_bit_scales(x, pairs):
    for name, t in pairs:
        if (t is not None) != (x.dtype == torch.float8_e4m3fn):
            raise ValueError("%s: 8-bit operands and their scales belong together" % name)


# ---------------------------------------------------------------- norm

def rms_norm(x, weight, residual=None, eps=1e-6, eight_bit=False, keep_rstd=False):
    """sum = x + residual, y = sum / sqrt(mean(sum^2) + eps) * weight for each row, of the sum ahead of its rounding.  float32, float16 or
    bfloat16; with ``eight_bit`` y is float8_e4m3fn and stands for y * scale[row].  ``keep_rstd`` keeps 1 / length of each row, which the
    backward pass reads together with ``sum``."""
    rows, ldx = _rows(x, "x", dtypes=_NORM_TYPES)
    columns, where = x.shape[-1], x.get_device()
    w = _vector(weight, "weight", columns, x.dtype, where)
    r, ldr, total = 0, 0, None
    if residual is not None:
        ldr = _rows(residual, "residual", shape=x.shape, dtypes=(x.dtype,))[1]
        r, total = _pointer(residual, "residual", where), _like(x, x.dtype)
    y = _like(x, torch.float8_e4m3fn if eight_bit else x.dtype)
    scale = _row_numbers(x, where) if eight_bit else None
    rstd = _row_numbers(x, where) if keep_rstd else None
    _call(_RMS_NORM, where, x.data_ptr(), r, w, y.data_ptr(), 0 if total is None else total.data_ptr(),
          scale.data_ptr() if eight_bit else 0, rstd.data_ptr() if keep_rstd else 0, rows, columns, ldx, ldr, eps, _TYPES[x.dtype], _TYPES[y.dtype])
    return RmsNorm(y, x if total is None else total, scale, rstd)


def rms_norm_backward(dy, sum, weight, rstd, dsum=None):
    """Gradients of ``rms_norm`` from the gradient of y and, where the sum is used further on, the gradient ``dsum`` of the sum."""
    rows, lds = _rows(sum, "sum", dtypes=_NORM_TYPES)
    columns, where = sum.shape[-1], sum.get_device()
    ldy = _rows(dy, "dy", shape=sum.shape, dtypes=(sum.dtype,))[1]
    w = _vector(weight, "weight", columns, sum.dtype, where)
    lengths = _row_scale(rstd, "rstd", sum, rows, where)
    d, ldd = 0, 0
    if dsum is not None:
        ldd = _rows(dsum, "dsum", shape=sum.shape, dtypes=(sum.dtype,))[1]
        d = _pointer(dsum, "dsum", where)
    dx = _like(sum, sum.dtype)
    dweight = weight.new_empty(columns)
    _call(_RMS_NORM_BACKWARD, where, _pointer(dy, "dy", where), sum.data_ptr(), w, lengths, d, dx.data_ptr(), dweight.data_ptr(), rows, columns,
          ldy, lds, ldd, _TYPES[sum.dtype])
    return RmsNormGradients(dx, dweight)


def quantize_rows(x):
    """x as float8_e4m3fn with a scale for each row, max|row| / 448 (1 for a row of zeros): weights once, activations where no norm
    precedes the product."""
    rows, ldx = _rows(x, "x", dtypes=_NORM_TYPES)
    q = _like(x, torch.float8_e4m3fn)
    scale = _row_numbers(x, x.get_device())
    _call(_QUANTIZE_ROWS, x.get_device(), x.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, x.shape[-1], ldx, _TYPES[x.dtype])
    return EightBitRows(q, scale)


# ---------------------------------------------------------------- linear

def _result_dtype(x, dtype):
    if x.dtype != torch.float8_e4m3fn:
        if dtype not in (None, x.dtype):
            raise ValueError("results of 16-bit operands are of their type, %s" % x.dtype)
        return x.dtype
    if dtype not in (None,) + _HALVES:
        raise ValueError("results of 8-bit operands are float16 or bfloat16")
    return dtype or torch.bfloat16


def linear(x, weight, bias=None, residual=None, activation="none", x_scale=None, weight_scale=None, dtype=None, keep_pre=False):
    """y = activation(x weight^T + bias) + residual.  x and weight are float16 or bfloat16, or float8_e4m3fn with ``x_scale`` (of each row
    of x) and ``weight_scale`` (of each output), then ``dtype`` (bfloat16) is the result's type.  bias and residual are of the result's
    type.  ``keep_pre`` keeps the sums ahead of the activation, which the backward pass reads."""
    rows, ldx = _rows(x, "x", dtypes=_PRODUCT_TYPES)
    k, where = x.shape[-1], x.get_device()
    ldw = _matrix(weight, "weight", None, k, x.dtype)
    n, out = weight.shape[0], _result_dtype(x, dtype)
    _eight_bit_scales(x, (("x_scale", x_scale), ("weight_scale", weight_scale)))
    shape = x.shape[:-1] + (n,)
    xs = 0 if x_scale is None else _row_scale(x_scale, "x_scale", x, rows, where)
    ws = 0 if weight_scale is None else _vector(weight_scale, "weight_scale", n, torch.float32, where)
    b = 0 if bias is None else _vector(bias, "bias", n, out, where)
    r, ldr = 0, 0
    if residual is not None:
        ldr = _rows(residual, "residual", shape=shape, dtypes=(out,))[1]
        r = _pointer(residual, "residual", where)
    if k == 0:
        rows = shape[:-1].numel()
    a = _activation(activation)
    y = _new(x, shape, out)
    pre = torch.empty_like(y) if keep_pre else None
    _call(_LINEAR, where, x.data_ptr(), _pointer(weight, "weight", where), b, r, xs, ws, y.data_ptr(), pre.data_ptr() if keep_pre else 0,
          rows, n, k, ldx, ldw, ldr, a, _TYPES[x.dtype], _TYPES[out])
    return Linear(y, pre)


def linear_backward(dy, x, weight, pre=None, activation="none", bias=False):
    """Gradients of ``linear`` (16-bit operands) of x, the weight and, where asked for, the bias.  ``pre``: what ``keep_pre`` kept, for any activation
    but "none".  The gradient of the residual is dy."""
    rows, ldx = _rows(x, "x", dtypes=_HALVES)
    k, where = x.shape[-1], x.get_device()
    ldw = _matrix(weight, "weight", None, k, x.dtype)
    n = weight.shape[0]
    shape = x.shape[:-1] + (n,)
    rows = shape[:-1].numel()
    ldy = _rows(dy, "dy", shape=shape, dtypes=(x.dtype,))[1]
    a, ldp = _activation(activation), 0
    if (pre is not None) != (activation != "none"):
        raise ValueError("pre: an activation and the sums ahead of it belong together")
    if pre is not None:
        ldp = _rows(pre, "pre", shape=shape, dtypes=(x.dtype,))[1]
    dx = _like(x, x.dtype)
    dweight = _like(weight, x.dtype)
    dbias = x.new_empty(n) if bias else None
    _call(_LINEAR_BACKWARD, where, _pointer(dy, "dy", where), x.data_ptr(), _pointer(weight, "weight", where), 0 if pre is None else _pointer(pre, "pre", where),
          dx.data_ptr(), dweight.data_ptr(), dbias.data_ptr() if bias else 0, rows, n, k, ldy, ldx, ldw, ldp, a, _TYPES[x.dtype])
    return LinearGradients(dx, dweight, dbias)


# ---------------------------------------------------------------- gated linear

def gated_linear(x, gate_weight, up_weight, activation="silu", x_scale=None, gate_scale=None, up_scale=None, dtype=None, keep_pre=False):
    """h = activation(x gate_weight^T) * (x up_weight^T), types and scales as for ``linear``.  ``keep_pre`` keeps both projections, which
    the backward pass reads."""
    rows, ldx = _rows(x, "x", dtypes=_PRODUCT_TYPES)
    k, where = x.shape[-1], x.get_device()
    ldg = _matrix(gate_weight, "gate_weight", None, k, x.dtype)
    n, out = gate_weight.shape[0], _result_dtype(x, dtype)
    ldu = _matrix(up_weight, "up_weight", n, k, x.dtype)
    _eight_bit_scales(x, (("x_scale", x_scale), ("gate_scale", gate_scale), ("up_scale", up_scale)))
    xs = 0 if x_scale is None else _row_scale(x_scale, "x_scale", x, rows, where)
    gs = 0 if gate_scale is None else _vector(gate_scale, "gate_scale", n, torch.float32, where)
    us = 0 if up_scale is None else _vector(up_scale, "up_scale", n, torch.float32, where)
    a, shape = _activation(activation), x.shape[:-1] + (n,)
    if k == 0:
        rows = shape[:-1].numel()
    h = _new(x, shape, out)
    gate, up = (torch.empty_like(h), torch.empty_like(h)) if keep_pre else (None, None)
    _call(_GATED_LINEAR, where, x.data_ptr(), _pointer(gate_weight, "gate_weight", where), _pointer(up_weight, "up_weight", where), xs, gs, us, h.data_ptr(),
          gate.data_ptr() if keep_pre else 0, up.data_ptr() if keep_pre else 0, rows, n, k, ldx, ldg, ldu, a, _TYPES[x.dtype], _TYPES[out])
    return GatedLinear(h, gate, up)


def gated_linear_backward(dh, x, gate_weight, up_weight, gate, up, activation="silu"):
    """Gradients of ``gated_linear`` (16-bit operands) of x and both weights; ``gate`` and ``up`` are what ``keep_pre`` kept."""
    rows, ldx = _rows(x, "x", dtypes=_HALVES)
    k, where = x.shape[-1], x.get_device()
    ldg = _matrix(gate_weight, "gate_weight", None, k, x.dtype)
    n = gate_weight.shape[0]
    ldu = _matrix(up_weight, "up_weight", n, k, x.dtype)
    shape = x.shape[:-1] + (n,)
    rows = shape[:-1].numel()
    ldh, ld_gate, ld_up = [_rows(t, name, shape=shape, dtypes=(x.dtype,))[1] for name, t in (("dh", dh), ("gate", gate), ("up", up))]
    a = _activation(activation)
    dx = _like(x, x.dtype)
    dg, du = _like(gate_weight, x.dtype), _like(up_weight, x.dtype)
    _call(_GATED_LINEAR_BACKWARD, where, _pointer(dh, "dh", where), x.data_ptr(), _pointer(gate_weight, "gate_weight", where), _pointer(up_weight, "up_weight", where),
          _pointer(gate, "gate", where), _pointer(up, "up", where), dx.data_ptr(), dg.data_ptr(), du.data_ptr(), rows, n, k, ldh, ldx, ldg, ldu, ld_gate, ld_up, a,
          _TYPES[x.dtype])
    return GatedLinearGradients(dx, dg, du)
