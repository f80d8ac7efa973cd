"""Products in 8-bit integers with a scale for each token and each output channel, for serving dense layers and shared experts.

A matrix [N,K] is (codes int8 [N,K], scales FP32 [N]), its values codes * scales; tokens [T,K] are (codes int8 [T,K], scales FP32 [T]),
as ``dense.rms_norm(..., quantize="int8")`` and ``quantize_tokens`` leave them.  Sums are taken in 32-bit integers and are exact.  The
reference has no counterpart of this module.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib, ops


class W8Weights(NamedTuple):
    codes: torch.Tensor
    scales: torch.Tensor


def quantize(weight: torch.Tensor) -> W8Weights:
    """Round a matrix [N,K] to 8 bits, each row (output channel) by its own largest magnitude.  Torch operations; done once."""
    if weight.ndim != 2:
        raise ValueError("weight must be [N, K]")
    w = weight.float()
    scales = (w.abs().amax(dim=1) / 127).clamp_min(1e-20)
    return W8Weights(torch.round(w / scales[:, None]).clamp(-127, 127).to(torch.int8).contiguous(), scales)


def dequantize(weights: W8Weights) -> torch.Tensor:
    """The matrix's values in FP32."""
    return weights.codes.float() * weights.scales[:, None]


def quantize_tokens(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [T,K], scales FP32 [T]) of x [T,K] (FP32, BF16 or FP16, K a multiple of 16): scale = max(|x|) / 127 of the token, codes
    rounded to nearest even."""
    done = _lib.host().quantize_tokens(x)  # the ordinary call, made natively
    return ops.quantize_tokens(x) if done is None else done


def matmul(x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], weights: W8Weights, *, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [T,K] times the matrix [N,K]: [T,N].

    x: FP32, BF16 or FP16, quantised in the call, or a pair of codes and scales.  ``dtype``: of the result, FP32, BF16 or FP16 (None: x's
    own, BF16 for a pair).  K is a multiple of 16, at most 65536."""
    done = _lib.host().w8_matmul(x, *weights, dtype)  # the ordinary call, made natively
    return ops.w8_matmul(x, *weights, dtype) if done is None else done
