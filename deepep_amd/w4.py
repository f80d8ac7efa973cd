"""Products of few tokens with weights held in 4 bits with group scales, for decode.

A matrix [N,K] is (packed uint8 [N,K/2], scales [N,K/group], zeros uint8 [N,K/group] or None); its values are
(q - zero) * scale, q two to a byte along K with the even k in the low nibble, zero 8 where none are given.  Experts' matrices carry
one more leading dimension.  Scales have the type of the rows that are multiplied, BF16 or FP16; a group is 32, 64 or a multiple
of 128 values.  Sums are taken in FP32 and rounded once.  The reference has no counterpart of this module: its experts are W4A8
(``deepep_amd.megamoe``, also for many tokens, from MXFP4 weights: it cannot read these).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib, ops


class W4Weights(NamedTuple):
    packed: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor] = None


def quantize(weight: torch.Tensor, group: int = 128, *, symmetric: bool = True, dtype: torch.dtype = torch.bfloat16) -> W4Weights:
    """Round a matrix [..., N, K] to 4 bits, each group of K by its own range, with scales in ``dtype``.  Torch operations; done once."""
    if not (group in (32, 64) or group > 0 and group % 128 == 0) or weight.shape[-1] % group:
        raise ValueError("group must be 32, 64 or a multiple of 128, and divide K")
    w = weight.float().unflatten(-1, (-1, group))
    zeros = None
    if symmetric:
        scales = (w.abs().amax(dim=-1) / 7).clamp_min(1e-7).to(dtype)
        shift = 8.0
    else:
        low, high = w.amin(dim=-1).clamp_max(0), w.amax(dim=-1).clamp_min(0)
        scales = ((high - low) / 15).clamp_min(1e-7).to(dtype)
        zeros = torch.round(-low / scales.float()).clamp(0, 15).to(torch.uint8)
        shift = zeros.float()[..., None]
    q = torch.round(w / scales.float()[..., None] + shift).clamp(0, 15).to(torch.uint8).flatten(-2)
    return W4Weights((q[..., 0::2] | (q[..., 1::2] << 4)).contiguous(), scales.contiguous(), zeros)


def dequantize(weights: W4Weights) -> torch.Tensor:
    """The matrix's values in FP32."""
    packed, scales, zeros = weights
    q = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float().unflatten(-1, (scales.shape[-1], -1))
    shift = 8.0 if zeros is None else zeros.float()[..., None]
    return ((q - shift) * scales.float()[..., None]).flatten(-2)


def matvec(x: torch.Tensor, weights: W4Weights, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [M,K] times the matrix [N,K]: [M,N] in x's type (BF16 or FP16).  ``out`` must overlap neither x nor the weights."""
    packed, scales, zeros = weights
    done = _lib.host().w4_matvec(x, packed, scales, zeros, out)  # the ordinary call, made natively
    return ops.w4_matvec(x, packed, scales, zeros, out=out) if done is None else done


def expert_ffn(x: torch.Tensor, topk_idx: torch.Tensor, topk_weights: torch.Tensor, gate_up: W4Weights, down: W4Weights, *,
               expert_begin: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The routed expert layer for few tokens: y[t] = sum over the slots of topk_weights[t,s] * down[e] (silu(gate) * up), gate and up
    the halves of gate_up[e] x[t], e = topk_idx[t,s] - expert_begin.

    x [T,H] BF16 or FP16, topk_idx int64 or int32 [T,K] (T * K at most 2048; -1 and experts that are not local do not count),
    topk_weights FP32 [T,K], gate_up [L,2I,H] (gate rows, then up rows), down [L,H,I].  Returns [T,H] in x's type; ``out`` may be x."""
    done = _lib.host().w4_experts(x, topk_idx, topk_weights, *gate_up, *down, expert_begin, out)  # the ordinary call, made natively
    if done is not None:
        return done
    return ops.w4_experts(x, topk_idx, topk_weights, gate_up, down, expert_begin, out)
