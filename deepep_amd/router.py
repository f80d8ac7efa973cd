"""The router of a mixture-of-experts layer: which experts a token goes to and with what weight, the balance loss over the batch's
sequences, and the gate's gradient.

    router = Router(256, 8, score="sigmoid", scale=2.5, num_groups=8, num_topk_groups=4)
    topk_idx, topk_weights, balance = router.route_with_balance(logits, bias, token_mask, sequence_offsets=offsets)
    ... buffer.dispatch(x, topk_idx=topk_idx, topk_weights=topk_weights, ...), experts, buffer.combine(...) and their backward ...
    grad_logits = router.backward(logits, topk_idx, topk_weights=topk_weights, grad_weights=grad_topk_weights,
                                  balance=balance, grad_losses=grad_losses)

Calls are queued on torch's current stream.  Nothing is recorded for autograd: the gradient is what ``backward`` returns, as with
``ElasticBuffer``.  The reference takes routes as given and has no counterpart of this module.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, ops


class BalanceLoss(NamedTuple):
    """``losses`` FP32 [B], one of each sequence (1 where its routes and probabilities are spread evenly); ``counts`` int32 [B,E],
    routes to each expert; ``tokens`` int32 [B], those with a route; and the offsets that cut the batch."""

    losses: torch.Tensor
    counts: torch.Tensor
    tokens: torch.Tensor
    sequence_offsets: Optional[torch.Tensor] = None


def _integer(name, value, lower, upper):
    if type(value) is not int or not lower <= value <= upper:
        raise ValueError(f"{name} must be an integer in [{lower}, {upper}]")


def _parameter(name):
    return property(lambda router: router._parameters[name])


class Router:
    """How a layer routes.

    ``score="softmax"``: experts are chosen by logit, weights are softmax probabilities.  ``score="sigmoid"``: chosen by
    sigmoid(logit) + bias, weights are the sigmoids.  An expert whose logit is -inf is never chosen.  ``normalize``: the chosen
    weights are divided by their sum; ``scale`` multiplies them.  ``num_groups`` > 1: the experts of the ``num_topk_groups`` best
    groups stay (a group's score: its largest key for softmax, the sum of its two largest for sigmoid).  Ties go to the lowest index.
    ``index_dtype``: int64 as ``ElasticBuffer.dispatch`` takes ids, or int32 as ``mega_moe`` does.  The parameters can be read and not set;
    a router can be copied and pickled.
    """

    num_experts, num_topk, num_groups, num_topk_groups, score, normalize, scale, index_dtype = map(_parameter, (
        "num_experts", "num_topk", "num_groups", "num_topk_groups", "score", "normalize", "scale", "index_dtype"))

    def __init__(self, num_experts: int, num_topk: int, *, score: str = "softmax", normalize: bool = True, scale: float = 1.0,
                 num_groups: int = 1, num_topk_groups: int = 1, index_dtype: torch.dtype = torch.int64):
        _integer("num_experts", num_experts, 1, 1024)
        _integer("num_topk", num_topk, 1, min(32, num_experts))
        _integer("num_groups", num_groups, 1, min(64, num_experts))
        _integer("num_topk_groups", num_topk_groups, 1, num_groups)
        if num_experts % num_groups:
            raise ValueError("num_groups must divide num_experts")
        if num_topk > num_experts // num_groups * num_topk_groups:
            raise ValueError("num_topk exceeds the experts of num_topk_groups groups")
        if score not in ops.SCORES:
            raise ValueError(f"score must be one of {ops.SCORES}")
        if not isinstance(scale, (int, float)) or not 1e-30 <= abs(scale) <= 1e30:
            raise ValueError("scale must be a number of 1e-30 to 1e30 in magnitude")
        if index_dtype not in (torch.int64, torch.int32):
            raise ValueError("index_dtype must be torch.int64 or torch.int32")
        self._parameters = dict(num_experts=num_experts, num_topk=num_topk, num_groups=num_groups, num_topk_groups=num_topk_groups, score=score,
                                normalize=bool(normalize), scale=float(scale), index_dtype=index_dtype)
        self._make_native()

    def _make_native(self):
        # Ordinary calls are made natively (csrc/host.cpp); the ones that come back as None, faulty or unusual, go through ops.
        self._native = _lib.host().Router(self.num_experts, self.num_topk, self.num_groups, self.num_topk_groups, ops.SCORES.index(self.score),
                                          int(self.normalize), self.scale, 8 if self.index_dtype == torch.int64 else 4)

    def __getstate__(self):
        return {name: value for name, value in self.__dict__.items() if name != "_native"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._make_native()

    def _spec(self) -> ops.RouterSpec:
        return ops.RouterSpec(self.num_experts, self.num_topk, self.num_groups, self.num_topk_groups, ops.SCORES.index(self.score),
                              int(self.normalize), self.scale, 0, 8)

    def _check_bias(self, bias):
        if bias is not None and self.score != "sigmoid":
            raise ValueError("a bias needs score='sigmoid'")

    def route(self, logits: torch.Tensor, bias: Optional[torch.Tensor] = None,
              token_mask: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(topk_idx [T,K], topk_weights FP32 [T,K])`` of ``logits`` [T,E] (FP32, BF16 or FP16), best first; -1 and 0 where fewer than
        K experts are left, and throughout for tokens that ``token_mask`` (bool [T]) has as False.  ``bias`` FP32 [E] takes part in the
        choice only."""
        self._check_bias(bias)
        done = self._native.route(logits, bias, token_mask)
        if done is not None:
            return done
        return ops.route(self._spec(), logits, bias, token_mask, self.index_dtype)

    def balance_loss(self, logits: torch.Tensor, topk_idx: torch.Tensor, sequence_offsets: Optional[torch.Tensor] = None) -> BalanceLoss:
        """Loss and counts of every sequence; ``sequence_offsets`` int32 [B+1] ascends from 0 to T (None: one sequence).  With c_e of a
        sequence's R routes on expert e and p the softmax of its N tokens' logits (sigmoid: the sigmoids over their sum), the loss is
        sum_e (E c_e / R) (sum_t p_te / N).  Tokens without a route are padding."""
        sums = self._native.balance_loss(logits, topk_idx, sequence_offsets)
        if sums is None:
            sums = ops.balance_loss(self._spec(), logits, topk_idx, sequence_offsets)
        return BalanceLoss(*sums, sequence_offsets)

    def route_with_balance(self, logits: torch.Tensor, bias: Optional[torch.Tensor] = None, token_mask: Optional[torch.Tensor] = None, *,
                           sequence_offsets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, BalanceLoss]:
        """``route`` and the ``balance_loss`` of its routes, in one pass over the logits."""
        self._check_bias(bias)
        done = self._native.route(logits, bias, token_mask, sequence_offsets)
        if done is None:
            done = ops.route_balance(self._spec(), logits, bias, token_mask, sequence_offsets, self.index_dtype)
        return done[0], done[1], BalanceLoss(done[2], done[3], done[4], sequence_offsets)

    def backward(self, logits: torch.Tensor, topk_idx: torch.Tensor, *, topk_weights: Optional[torch.Tensor] = None,
                 grad_weights: Optional[torch.Tensor] = None, balance: Optional[BalanceLoss] = None,
                 grad_losses: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Gradient of ``logits`` in their type.  ``grad_weights`` FP32 [T,K]: of the route weights (``combine`` returns it), with the
        ``topk_weights`` of ``route`` where they are normalised.  ``grad_losses`` FP32 [B] with ``balance``: of the balance losses.
        Either, or both in one pass.  The choice and the counts have no gradient."""
        if (balance is None) != (grad_losses is None):
            raise ValueError("balance and grad_losses belong together")
        offsets, counts, tokens = (None, None, None) if balance is None else (balance.sequence_offsets, balance.counts, balance.tokens)
        grad = self._native.backward(logits, topk_idx, topk_weights, grad_weights, offsets, counts, tokens, grad_losses)
        if grad is not None:
            return grad
        return ops.router_backward(self._spec(), logits, topk_idx, topk_weights, grad_weights, offsets, counts, tokens, grad_losses)
