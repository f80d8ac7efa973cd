"""What every token of a layer passes through beside the routed experts: the root-mean-square norm with the residual's addition and an
output in 8 bits, and the gated feed-forward block of shared experts and dense layers, both with their gradients.

    normed = rms_norm(x, weight, residual, quantize="fp8")       # normed.codes, normed.scales go into ElasticBuffer.dispatch as a pair
    y, kept = gated_ffn(normed.y, gate_up, down, keep=True)
    grad_normed, grad_gate_up, grad_down = gated_ffn_backward(grad_y, normed.y, gate_up, down, kept)
    grad_x, grad_weight = rms_norm_backward(grad_normed, normed.stream, weight, normed.rstd, grad_stream)

Calls are queued on torch's current stream.  Nothing is recorded for autograd: gradients are what the ``backward`` functions return, as
with ``ElasticBuffer`` and ``Router``.  The reference has no counterpart of this module.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib, ops


class Norm(NamedTuple):
    """``y`` [T,H] in x's type (None if it was not asked for); ``stream`` [T,H], what was normed: x itself, or x + residual in x's type;
    ``rstd`` FP32 [T]; ``codes`` and ``scales`` where the output was quantised, else None."""

    y: Optional[torch.Tensor]
    stream: torch.Tensor
    rstd: torch.Tensor
    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
             quantize: Optional[str] = None, output: bool = True) -> Norm:
    """weight * s / sqrt(mean(s^2) + eps) of every row of s = x + residual (rounded to x's type; x itself without a residual).

    x, residual [T,H] FP32, BF16 or FP16, H a multiple of 8 up to 16384; weight [H] in x's type or FP32.  ``quantize``, from FP32 values:
    ``"fp8"`` codes float8_e4m3fn [T,H] and FP32 scales [T, ceil(H/128)], as ``ElasticBuffer.dispatch`` takes them (H a multiple of 16);
    ``"mxfp8"`` codes float8_e4m3fn and e8m0 bytes uint8 [T,H/32], as ``fp8_fp4_mega_moe`` takes them (H a multiple of 32);
    ``"int8"`` codes int8 and FP32 scales [T], as ``w8.matmul`` takes them (H a multiple of 16).  ``output=False``: y is not stored.

    Squares are added up in FP32: values from 1.8e19 / sqrt(H) on, whose sum passes its range, are normed to 0."""
    done = _lib.host().rms_norm(x, weight, residual, eps, quantize, output)  # the ordinary call, made natively
    if done is None:
        done = ops.rms_norm(x, weight, residual, eps, quantize, output)
    y, stream, rstd, codes, scales = done
    return Norm(y, x if stream is None else stream, rstd, codes, scales)


def rms_norm_backward(grad_y: torch.Tensor, stream: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      grad_stream: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(grad_x [T,H] in x's type, grad_weight FP32 [H])`` from the gradient of ``y`` and, optional, that which reaches ``stream`` from
    elsewhere.  grad_x is the gradient of x and of the residual alike.  Sums repeat bit for bit."""
    done = _lib.host().rms_norm_backward(grad_y, stream, weight, rstd, grad_stream)  # the ordinary call, made natively
    return ops.rms_norm_backward(grad_y, stream, weight, rstd, grad_stream) if done is None else done


def gated_ffn(x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, *,
              keep: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """(silu(gate) * up) down^T, gate and up the halves of x gate_up^T.

    x [T,H] BF16 or FP16, gate_up [2I,H] (gate rows, then up rows), down [H,I], H and I multiples of 8.  Returns [T,H] in x's type; with
    ``keep`` also what ``gated_ffn_backward`` needs (FP32 [T,2I], the products before the activation).  Sums are taken in FP32; the rows
    between the products are rounded to x's type."""
    done = _lib.host().gated_ffn(x, gate_up, down, keep)  # the ordinary call, made natively
    return ops.gated_ffn(x, gate_up, down, keep) if done is None else done


def gated_ffn_backward(grad_y: torch.Tensor, x: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor,
                       kept: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(grad_x, grad_gate_up, grad_down)`` in x's type from the gradient of the output; ``kept`` as ``gated_ffn`` returned it for these x
    and gate_up.  Sums repeat bit for bit."""
    done = _lib.host().gated_ffn_backward(grad_y, x, gate_up, down, kept)  # the ordinary call, made natively
    return ops.gated_ffn_backward(grad_y, x, gate_up, down, kept) if done is None else done
