"""The operators of a transformer's feed-forward sublayer on torch tensors: the residual stream's addition and root-mean-square norm, the matrix
product with bias, activation and residual in its epilogue, and both projections of a gated feed-forward layer in one
kernel; each with its backward pass, on 16-bit operands or (forward) 8-bit ones with scales.  For a sublayer with experts: a router's choice, the products of
rows that are grouped by expert, and the weighted sum of a token's rows, with their backward passes.  For serving: products with weights in 4 bits.

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


class Route(NamedTuple):
    experts: torch.Tensor                   # [..., k] int32: the chosen ones, the best first; -1: none was left
    weights: torch.Tensor                   # [..., k] float32
    offsets: torch.Tensor                   # [experts + 1] int32: where each expert's places begin, and the last one's end
    rows: torch.Tensor                      # [tokens k] int32: the token of each place, -1 behind the last
    places: torch.Tensor                    # [..., k] int32: the place of each choice, -1 where there is none


class GroupedLinearGradients(NamedTuple):
    dx: torch.Tensor                        # of each place
    dweight: torch.Tensor


class GroupedGatedLinearGradients(NamedTuple):
    dx: torch.Tensor                        # of each place
    dgate_weight: torch.Tensor
    dup_weight: torch.Tensor


class CombineGradients(NamedTuple):
    dx: torch.Tensor
    dweights: Optional[torch.Tensor] = None


class FourBitRows(NamedTuple):
    q: torch.Tensor                         # [..., (columns + 1) // 2] uint8: two values to a byte, the first in the low half
    scale: torch.Tensor                     # [..., (columns + 31) // 32] uint8: exponent and 127 of the power of two of each 32


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


# ---------------------------------------------------------------- experts

def route(logits, k, normalise=True):
    """The k largest of each row of a router's logits (float32, float16 or bfloat16; ties go to the lowest index, minus infinity is never chosen, NaN before all),
    their weights -- the softmax over the chosen ones, or without ``normalise`` over all --, and the places of the rows grouped by expert, in the order of the
    tokens: ``rows`` and ``offsets`` are what the grouped products take, ``places`` and ``weights`` what ``combine`` takes.  Tokens whose logits are all minus infinity (padding) have no
    place; as many places at the end are empty.  At most 1024 experts, 16 choices.  Nothing of it is read by the host."""
    return Route(*_operators.route(logits, k, normalise))


def route_backward(dweights, logits, experts, normalise=True):
    """Gradient of the logits from that of ``route``'s weights; ``experts`` are its choices."""
    return _operators.route_backward(dweights, logits, experts, normalise)[0]


def grouped_linear(x, weight, offsets, rows=None, x_scale=None, weight_scale=None, dtype=None):
    """y[s] = x[s] weight[g]^T for the places s from offsets[g] to offsets[g + 1] (int32, on the GPU), with weight [groups, N, K] and the types of ``linear``
    (``weight_scale`` [groups, N]).  With ``rows`` place s takes the row x[rows[s]] instead, and the result has a row for each of ``rows``.  Places ahead of the first
    group's and behind the last one's, and those whose number is none of x's, are rows of zeros, whatever weights and scales hold; so ``weight[a:b]`` with ``offsets[a:b + 1]`` are the results of these groups alone."""
    return _operators.grouped_linear(x, weight, offsets, rows, x_scale, weight_scale, _result_type(dtype))[0]


def grouped_linear_backward(dy, x, weight, offsets, rows=None):
    """Gradients of ``grouped_linear`` (16-bit operands): dx of each place (with ``rows`` the gradient of x is ``combine(dx, places)``) and of the weights, zeros for
    a group without places.  A place whose number is none of x's counts as dy times zeros there."""
    return GroupedLinearGradients(*_operators.grouped_linear_backward(dy, x, weight, offsets, rows))


def grouped_gated_linear(x, gate_weight, up_weight, offsets, rows=None, activation="silu", x_scale=None, gate_scale=None, up_scale=None, dtype=None, keep_pre=False):
    """``gated_linear`` for rows grouped like those of ``grouped_linear``."""
    return GatedLinear(*_operators.grouped_gated_linear(x, gate_weight, up_weight, offsets, rows, _activation(activation), x_scale, gate_scale, up_scale, _result_type(dtype), keep_pre))


def grouped_gated_linear_backward(dh, x, gate_weight, up_weight, gate, up, offsets, rows=None, activation="silu"):
    """Gradients of ``grouped_gated_linear`` (16-bit operands): dx of each place, and both weights; ``gate`` and ``up`` are what ``keep_pre`` kept."""
    return GroupedGatedLinearGradients(*_operators.grouped_gated_linear_backward(dh, x, gate_weight, up_weight, gate, up, offsets, rows, _activation(activation)))


def combine(x, places, weights=None, residual=None):
    """y[t] = residual[t] + the sum over j of weights[t, j] x[places[t, j]]: x [places, N] float16 or bfloat16, ``places`` [..., k] int32 (numbers outside of x count as none),
    ``weights`` float32 (without: ones)."""
    return _operators.combine(x, places, weights, residual)[0]


def combine_backward(dy, x, places, weights, rows):
    """Gradients of ``combine``: of x, and of the weights where there are some (None: ones).  Each place is in ``places`` once at most; ``rows``, the token of each place, is that of
    the route: a place that is no token's, or that its token's ``places`` have left out since, has a gradient of zeros."""
    return CombineGradients(*_operators.combine_backward(dy, x, places, weights, rows))


# ---------------------------------------------------------------- 4-bit weights

def quantize_groups(x):
    """x (float32, float16 or bfloat16) in 4 bits: values of e2m1 -- 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives, to the nearest -- and for each 32 of a row the smallest
    power of two by which the largest of them is at most 6 (1 for zeros; NaN, 255, where one of them is not finite)."""
    return FourBitRows(*_operators.quantize_groups(x))


def four_bit_linear(x, weight, weight_scale, bias=None, residual=None, activation="none"):
    """``linear`` with a weight in 4 bits (``quantize_groups``' values and scales); x, bias and residual float16 or bfloat16.  Weights are multiplied as numbers of x's type, which are exact in
    bfloat16 below 2^128 and in float16 within its range, and infinite beyond."""
    return Linear(*_operators.four_bit_linear(x, weight, weight_scale, bias, residual, _activation(activation)))


def four_bit_gated_linear(x, gate_weight, up_weight, gate_scale, up_scale, activation="silu"):
    """``gated_linear`` with both weights in 4 bits."""
    return GatedLinear(*_operators.four_bit_gated_linear(x, gate_weight, up_weight, gate_scale, up_scale, _activation(activation)))


_operators = _native()
