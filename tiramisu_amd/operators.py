"""The operators of a transformer's feed-forward sublayer on torch tensors: the residual stream's addition and root-mean-square norm, the matrix
product with bias, activation and residual in its epilogue, and both projections of a gated feed-forward layer in one
kernel; each with its backward pass, on 16-bit operands or (forward) 8-bit ones with scales.

These functions check their arguments, allocate the results and call the runtime's C ABI (include/tiramisu_hip_wrappers.h), whose
kernels run on torch's current stream of the tensors' device; nothing waits for them.  They record nothing for autograd: the backward passes are
functions of their own, and tensors that require a gradient are taken where none is recorded (torch.no_grad()).  Leading dimensions are tokens: x of shape
[..., K] gives a result of shape [..., N].  Weights are [outputs, inputs].  Tensors need dense rows (stride 1 in the last
dimension), with one stride from row to row; others are refused, never copied silently.  Results are new, dense tensors.
ValueError says what does not fit, RuntimeError that the runtime refused the call (its reason is on stderr), torch's out-of-memory error that there is no
memory for results or scratch.  Scratch is torch's memory too: it is back with torch's allocator behind the call, and in a recorded graph it belongs to the graph, so
graphs may be replayed beside each other.
"""
import os
from typing import NamedTuple, Optional

import torch

from . import build as _build
from . import runtime as _runtime

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_RESULT_TYPES = {None: 0, torch.float16: 1, torch.bfloat16: 2}


def _native():
    """The extension that checks, allocates and calls (csrc/torch_operators.cpp), loaded against the runtime's library."""
    if not os.path.exists(_build.torch_module()):
        raise RuntimeError("%s is missing: run __graft_entry__.build() first" % _build.torch_module())
    _runtime.wrappers()
    from . import _torch_operators
    return _torch_operators


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


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation %r: one of %s" % (name, ", ".join(ACTIVATIONS)))
    return ACTIVATIONS[name]


def _result_type(dtype):
    if dtype not in _RESULT_TYPES:
        raise ValueError("results are float16 or bfloat16, not %s" % dtype)
    return _RESULT_TYPES[dtype]


# ---------------------------------------------------------------- norm

def rms_norm(x, weight, residual=None, eps=1e-6, eight_bit=False, keep_rstd=False):
    """sum = x + residual, y = sum / sqrt(mean(sum^2) + eps) * weight for each row, of the sum ahead of its rounding.  float32, float16 or
    bfloat16; with ``eight_bit`` y is float8_e4m3fn and stands for y * scale[row].  ``keep_rstd`` keeps 1 / length of each row, which the
    backward pass reads together with ``sum``."""
    y, total, scale, rstd = _operators.rms_norm(x, weight, residual, eps, eight_bit, keep_rstd)
    return RmsNorm(y, x if total is None else total, scale, rstd)


def rms_norm_backward(dy, sum, weight, rstd, dsum=None):
    """Gradients of ``rms_norm`` from the gradient of y and, where the sum is used further on, the gradient ``dsum`` of the sum."""
    return RmsNormGradients(*_operators.rms_norm_backward(dy, sum, weight, rstd, dsum))


def quantize_rows(x):
    """x as float8_e4m3fn with a scale for each row, max|row| / 448 (1 where that is zero, and for a row of no elements): weights once, activations where no norm
    precedes the product."""
    return EightBitRows(*_operators.quantize_rows(x))


# ---------------------------------------------------------------- linear

def linear(x, weight, bias=None, residual=None, activation="none", x_scale=None, weight_scale=None, dtype=None, keep_pre=False):
    """y = activation(x weight^T + bias) + residual.  x and weight are float16 or bfloat16, or float8_e4m3fn with ``x_scale`` (of each row
    of x) and ``weight_scale`` (of each output), then ``dtype`` (bfloat16) is the result's type.  bias and residual are of the result's
    type.  ``keep_pre`` keeps the sums ahead of the activation, which the backward pass reads."""
    return Linear(*_operators.linear(x, weight, bias, residual, _activation(activation), x_scale, weight_scale, _result_type(dtype), keep_pre))


def linear_backward(dy, x, weight, pre=None, activation="none", bias=False):
    """Gradients of ``linear`` (16-bit operands) of x, the weight and, where asked for, the bias.  ``pre``: what ``keep_pre`` kept, for any activation
    but "none".  The gradient of the residual is dy."""
    return LinearGradients(*_operators.linear_backward(dy, x, weight, pre, _activation(activation), bias))


# ---------------------------------------------------------------- gated linear

def gated_linear(x, gate_weight, up_weight, activation="silu", x_scale=None, gate_scale=None, up_scale=None, dtype=None, keep_pre=False):
    """h = activation(x gate_weight^T) * (x up_weight^T), types and scales as for ``linear``.  ``keep_pre`` keeps both projections, which
    the backward pass reads."""
    return GatedLinear(*_operators.gated_linear(x, gate_weight, up_weight, _activation(activation), x_scale, gate_scale, up_scale, _result_type(dtype), keep_pre))


def gated_linear_backward(dh, x, gate_weight, up_weight, gate, up, activation="silu"):
    """Gradients of ``gated_linear`` (16-bit operands) of x and both weights; ``gate`` and ``up`` are what ``keep_pre`` kept."""
    return GatedLinearGradients(*_operators.gated_linear_backward(dh, x, gate_weight, up_weight, gate, up, _activation(activation)))


_operators = _native()
