"""Microscaled 4-bit (MXFP4) operators: quantise rows, read them back, dense layers on the 4-bit matrix pipe, forward and
backward.  No counterpart in the reference, which is fp32 throughout.

A row is cut into blocks of 32 values; a block holds one power-of-two scale and 32 codes of 4 bits (0 .5 1 1.5 2 3 4 6 and
their negatives), so a value takes 4.25 bits.  The scale is 2^(floor(log2(largest magnitude)) - 2): the largest value lands
in [4, 8) of the code's range, what is above 6 saturates, everything else is rounded to nearest, ties to even.  A block that
holds a NaN or an infinity stands for NaN as a whole.

    q = mx.quantize(w)                      # MXTensor(codes, scales, K), 3.76 times smaller than bf16
    y = mx.linear(x, q, b)                  # serving: x is rounded on the call, q stays packed
    y = mx.linear(x, w, b, mx.ACT_SIN)      # training: w is a float tensor, gradients go straight through the rounding
    w = mx.dequantize(q, torch.bfloat16)    # the values the codes stand for

All of them run on the current stream of the tensors' device, allocate their outputs and workspaces from torch's allocator
and can be captured into a graph (with gradients: torch.autograd.grad inside the capture, after a warm-up on another stream, and
with no result of an eager pass over the same leaves still alive: it holds the leaves' autograd nodes on the eager stream, and a
capture that has to wait for that ends the process).
K is at most 2^22 and a matrix of packed rows below 2^32 groups of eight values (rows * 16 * ceil(K / 128)); a product takes
weights of up to 2^22 rows, a call that trains up to 65535 * 64 rows of x and of the weight.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _hip
from ._hip import ACT_NONE, ACT_RELU, ACT_SIGMOID, ACT_SIN
from .ops import MXLinearFunction

ACTIVATIONS = {"none": ACT_NONE, "relu": ACT_RELU, "sin": ACT_SIN, "sigmoid": ACT_SIGMOID}


class MXTensor(NamedTuple):
    """Packed rows of K values: codes uint8 [rows, 64 ceil(K/128)] (low nibble = even index), scales uint8
    [rows, 4 ceil(K/128)] (a block's scale is 2^(s - 127), 255 = NaN); zeros behind K."""
    codes: Tensor
    scales: Tensor
    K: int

    @property
    def rows(self) -> int:
        return self.codes.shape[0]


def _matrix(x: Tensor, name: str) -> Tensor:
    """[.., K] as a matrix with contiguous rows; a view where the layout allows it."""
    if x.dim() == 2 and x.is_contiguous() and x.shape[1]:
        return x
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: expected rows of at least one value, got shape {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def quantize(x: Tensor) -> MXTensor:
    """Packed rows of x [.., K] (float32, bfloat16, float16; leading dimensions are flattened).  Not differentiable: the
    gradient of a layer goes through `linear`."""
    m = _matrix(x, "x")
    return MXTensor(*_hip.mx_quantize(m), m.shape[1])


def dequantize(q: MXTensor, dtype: torch.dtype = torch.float32) -> Tensor:
    """[rows, K] values of packed rows, rounded once to `dtype` (exact in float32 and bfloat16)."""
    return _hip.mx_dequantize(q.codes, q.scales, q.K, dtype)


def linear(x: Tensor, weight: Union[MXTensor, Tensor], bias: Optional[Tensor] = None, act: int = ACT_NONE, pre: float = 1.0,
           post: float = 1.0) -> Tensor:
    """post * f(pre * (Q(x) Q(W)^T + bias)) for x [.., K] and a weight of N rows of K values -> [.., N], type of x.

    weight: packed rows (MXTensor), or a float tensor [N,K] of x's type that the call quantises.  act: ACT_NONE, ACT_RELU,
    ACT_SIN or ACT_SIGMOID.  Differentiable in x, a float weight and the bias: the gradients of the product at the rounded
    operands, straight through the rounding (first order, reverse mode only: a tangent of forward-mode differentiation is
    refused)."""
    if isinstance(weight, MXTensor):
        K, N, packed, W = weight.K, weight.rows, (weight.codes, weight.scales), None
    else:
        if weight.dim() != 2:
            raise ValueError(f"weight: expected [N,K], got shape {tuple(weight.shape)}")
        if weight.dtype != x.dtype or weight.device != x.device:
            raise TypeError(f"weight: expected {x.dtype} on {x.device} like x, got {weight.dtype} on {weight.device}")
        N, K = weight.shape
        packed, W = None, _matrix(weight, "weight")
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not end with the weight's {K} values per row")
    if act not in (ACT_NONE, ACT_RELU, ACT_SIN, ACT_SIGMOID):
        raise ValueError(f"unknown activation {act}")
    if forward_ad._current_level >= 0:      # inside a dual_level; tangents do not show in requires_grad
        for t in (x, W, bias):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("mx.linear has no forward-mode derivative")
    m = _matrix(x, "x")
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (W is not None and W.requires_grad) or (bias is not None and bias.requires_grad)):
        y = MXLinearFunction.apply(m, W, packed, bias, act, float(pre), float(post))
    else:
        if packed is None:
            packed = _hip.mx_quantize(W)
        y = _hip.mx_linear_fwd(m, *packed, bias, act, pre, post)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)
