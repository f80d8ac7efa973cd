"""The operators around dispatch and combine that a mixture-of-experts layer needs, as cases that can be timed one by one.

Four families:

  route    the router: scores, group-limited top-k, route weights; with "backward" also the logits' gradient from the weight
           gradients that combine returns, with "balance" the balance loss beside it and one backward pass for both
  balance  the balance loss over sequences and the per-expert counts, given the routes; with "backward" its gradient
  matvec   products of a few rows with one matrix held in 4 bits with group scales
  experts  the expert layer for a few tokens: gate and up products, SwiGLU, down product and route-weighted sum over 4-bit weights

`own` says whose code computes them: this package's kernels, or (False) elementary torch operations in 32 bits, which run on a tree
that lacks the kernels.  Sizes are those of this repository's benchmark, protocol presets and tests, and generic ones beside them.
"""

from __future__ import annotations

import math

import torch

own = False

# Upper bounds of a drawn case, so that none costs more than the largest listed one.
_MOST_LOGITS = 65536 * 256
_MOST_ROUTED_WEIGHTS = 128 * 3 * 2048 * 7168  # routes * weights of an expert (the plain form widens each route's weights)
_MOST_HELD_WEIGHTS = 256 * 3 * 2048 * 7168    # experts * weights of an expert
_MOST_MATVEC = 64 * 8192 * 8192


def listed():
    return [
        # The smallest call: the router of one decoded token in a layer of 256 experts in eight groups. Launch and host time only.
        dict(name="route 1x256 grouped", family="route", tokens=1, experts=256, topk=8, score="sigmoid", normalize=True, scale=2.5,
             groups=8, topk_groups=4, bias=True, dtype="fp32", index="int64", padding=0.0, closed=0, backward=False, balance=False,
             sequences=1),
        # A decode batch in front of the W4A8 layer, which takes 32-bit ids; BF16 logits hold many ties.
        dict(name="route 128x384 bf16", family="route", tokens=128, experts=384, topk=6, score="softmax", normalize=True, scale=1.0,
             groups=1, topk_groups=1, bias=False, dtype="bf16", index="int32", padding=0.0, closed=0, backward=False, balance=False,
             sequences=1),
        # A training chunk with padding tokens, sizes that are no powers of two, two experts out of service; weights that are
        # not normalised, so that every logit has a gradient.
        dict(name="route train 1000x160 masked", family="route", tokens=1000, experts=160, topk=6, score="softmax", normalize=False,
             scale=1.0, groups=1, topk_groups=1, bias=False, dtype="bf16", index="int64", padding=0.15, closed=2, backward=True,
             balance=False, sequences=1),
        # A training step's routing of 4096 tokens over 128 experts: both directions, no balance loss (the bias does that).
        dict(name="route train 4096x128", family="route", tokens=4096, experts=128, topk=8, score="sigmoid", normalize=True, scale=1.0,
             groups=1, topk_groups=1, bias=True, dtype="fp32", index="int64", padding=0.0, closed=0, backward=True, balance=False,
             sequences=1),
        # The largest: a whole batch through router and balance loss, forward and backward, 16 sequences of uneven length.
        dict(name="step 65536x256 grouped", family="route", tokens=65536, experts=256, topk=8, score="sigmoid", normalize=True,
             scale=2.5, groups=8, topk_groups=4, bias=True, dtype="fp32", index="int64", padding=0.05, closed=0, backward=True,
             balance=True, sequences=16),
        # The counts and the loss alone, as an evaluation or a monitor of the bias update takes them.
        dict(name="balance 777x32", family="balance", tokens=777, experts=32, topk=4, score="softmax", dtype="fp32", index="int64",
             padding=0.0, closed=0, sequences=1, backward=False),
        # A training batch's loss and its gradient over sequences of uneven length, BF16 logits.
        dict(name="balance train 16384x160 ragged", family="balance", tokens=16384, experts=160, topk=6, score="softmax", dtype="bf16",
             index="int64", padding=0.15, closed=2, sequences=7, backward=True),
        # One decoded token through a shared expert's gate and up matrices.
        dict(name="matvec 1x7168 to 4096", family="matvec", rows=1, inputs=7168, outputs=4096, group=128, zeros=False, dtype="bf16"),
        # A speculative batch through a matrix whose sizes are no whole tiles, zero points and short groups.
        dict(name="matvec 33x2880 to 1407", family="matvec", rows=33, inputs=2880, outputs=1407, group=32, zeros=True, dtype="fp16"),
        # One token through its 8 of 256 experts: nothing but the stream of their weights.
        dict(name="experts 1x7168 of 256", family="experts", tokens=1, hidden=7168, inter=2048, topk=8, experts=256, group=128,
             zeros=False, dtype="bf16", masked=0.0, skew=0.0),
        # A few tokens of a smaller model, two of their routes elsewhere, sizes that are no whole tiles.
        dict(name="experts 5x2880 of 32", family="experts", tokens=5, hidden=2880, inter=1408, topk=4, experts=32, group=64,
             zeros=True, dtype="fp16", masked=0.1, skew=0.0),
        # The largest decode batch here: about a hundred experts are touched, some by several tokens.
        dict(name="experts 16x7168 of 256", family="experts", tokens=16, hidden=7168, inter=2048, topk=8, experts=256, group=128,
             zeros=False, dtype="bf16", masked=0.0, skew=0.6),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _multiple(rng, step, low, high):
    return _log_int(rng, -(-low // step), high // step) * step


def draw(rng):
    family = rng.choices(("route", "balance", "matvec", "experts"), weights=(4, 3, 3, 3))[0]
    while True:
        if family in ("route", "balance"):
            groups = rng.choice((1, 1, 2, 4, 8)) if family == "route" else 1
            experts = groups * _log_int(rng, max(1, 8 // groups), 512 // groups)
            topk_groups = rng.randint(1, groups)
            topk = rng.randint(1, 10)
            case = dict(family=family, tokens=_log_int(rng, 1, 65536), experts=experts, topk=topk,
                        score=rng.choice(("softmax", "sigmoid")), dtype=rng.choice(("fp32", "fp32", "bf16")),
                        index=rng.choice(("int64", "int64", "int32")), padding=rng.choice((0.0, 0.0, 0.15)), closed=rng.choice((0, 0, 0, 2)),
                        sequences=rng.choice((1, 1, _log_int(rng, 2, 64))), backward=rng.random() < 0.6)
            if family == "route":
                case.update(normalize=rng.random() < 0.7, scale=rng.choice((1.0, 1.0, 2.5)), groups=groups, topk_groups=topk_groups,
                            bias=case["score"] == "sigmoid" and rng.random() < 0.7, balance=case["backward"] and rng.random() < 0.4)
            if case["tokens"] * experts <= _MOST_LOGITS and topk + case["closed"] <= experts // groups * topk_groups:
                return case
        elif family == "matvec":
            group = rng.choice((32, 64, 128))
            case = dict(family=family, rows=_log_int(rng, 1, 64), inputs=_multiple(rng, group, 256, 8192), outputs=_log_int(rng, 64, 8192),
                        group=group, zeros=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "fp16")))
            if case["rows"] * case["inputs"] * case["outputs"] <= _MOST_MATVEC:
                return case
        else:
            group = rng.choice((32, 64, 128))
            case = dict(family=family, tokens=_log_int(rng, 1, 64), hidden=_multiple(rng, group, 512, 7168),
                        inter=_multiple(rng, group, 256, 4096), topk=rng.randint(1, 8), experts=_log_int(rng, 8, 256), group=group,
                        zeros=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "fp16")), masked=rng.choice((0.0, 0.0, 0.15)),
                        skew=rng.choice((0.0, 0.6)))
            weights = 3 * case["inter"] * case["hidden"]
            if case["tokens"] * case["topk"] * weights <= _MOST_ROUTED_WEIGHTS and case["experts"] * weights <= _MOST_HELD_WEIGHTS:
                return case


# ---- inputs ------------------------------------------------------------------------------------------------------------------
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_INDEX = {"int64": torch.int64, "int32": torch.int32}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _logits(case, gen):
    """A gate's logits: tokens' own preferences over experts of uneven popularity; experts out of service are -inf."""
    tokens, experts = case["tokens"], case["experts"]
    z = torch.randn((tokens, experts), generator=gen, device="cuda") + 0.5 * torch.randn((experts,), generator=gen, device="cuda")
    if case["closed"]:
        z[:, torch.randperm(experts, generator=gen, device="cuda")[: case["closed"]]] = -math.inf
    return z.to(_DTYPES[case["dtype"]])


def _padding(case, gen):
    """[T] which tokens are real, or None where all are."""
    if not case["padding"]:
        return None
    real = torch.ones((case["tokens"],), dtype=torch.bool, device="cuda")
    real[torch.randperm(case["tokens"], generator=gen, device="cuda")[: int(case["padding"] * case["tokens"])]] = False
    return real


def _sequence_offsets(case, gen):
    """[B+1] where the batch's sequences begin, of uneven length, or None for one sequence."""
    if case["sequences"] == 1:
        return None
    cuts = torch.randint(0, case["tokens"] + 1, (case["sequences"] - 1,), generator=gen, device="cuda").sort().values
    ends = torch.tensor([0, case["tokens"]], device="cuda")
    return torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)


def _w4(gen, experts, n, k, group, zeros, dtype):
    """Normal weights of scale 0.02 as 4-bit codes: each byte's two codes are drawn from the codes' own distribution."""
    quantiles = torch.special.ndtri((torch.arange(256, device="cuda", dtype=torch.float32) + 0.5) / 256) * 2.7
    codes = torch.clamp(torch.round(quantiles) + 8, 0, 15).to(torch.uint8)
    table = (codes[None, :] | (codes[:, None] << 4)).reshape(-1)
    packed = torch.empty((experts, n, k // 2), dtype=torch.uint8, device="cuda")
    for e in range(experts):
        packed[e] = table[torch.randint(0, 65536, (n, k // 2), generator=gen, device="cuda", dtype=torch.int32)]
    scales = (0.0074 * (0.7 + 0.6 * torch.rand((experts, n, k // group), generator=gen, device="cuda"))).to(dtype)
    points = None
    if zeros:
        points = torch.randint(6, 11, (experts, n, k // group), generator=gen, device="cuda", dtype=torch.uint8)
    return packed, scales, points


def _expert_routes(gen, case):
    """Distinct top-k experts per token, expert e with popularity (e + 1)^-skew; a share of the routes is served elsewhere (-1)."""
    tokens, experts, topk = case["tokens"], case["experts"], case["topk"]
    popularity = -case["skew"] * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    uniform = torch.rand((tokens, experts), generator=gen, device="cuda").clamp_(1e-20, 1.0 - 1e-7)
    idx = (popularity - torch.log(-torch.log(uniform))).topk(topk, dim=1).indices
    elsewhere = int(case["masked"] * tokens * topk)
    if elsewhere:
        idx.view(-1)[torch.randperm(tokens * topk, generator=gen, device="cuda")[:elsewhere]] = -1
    return idx.contiguous()


class _State:
    def __init__(self, case, **fields):
        self.case = case
        self.router = None  # the package's router, made at the first pass that uses it and kept, as a layer keeps it
        self.__dict__.update(fields)


def prepare(case, seed):
    gen = _generator(seed)
    family = case["family"]
    if family == "route":
        tokens, experts, topk = case["tokens"], case["experts"], case["topk"]
        return _State(
            case, logits=_logits(case, gen), bias=0.05 * torch.randn((experts,), generator=gen, device="cuda") if case["bias"] else None,
            real=_padding(case, gen), offsets=_sequence_offsets(case, gen) if case["balance"] else None,
            grad_weights=torch.randn((tokens, topk), generator=gen, device="cuda") if case["backward"] else None,
            grad_losses=1e-3 * (1.0 + torch.rand((case["sequences"],), generator=gen, device="cuda")) if case["balance"] else None)
    if family == "balance":
        logits = _logits(case, gen)
        idx = logits.float().topk(case["topk"], dim=1).indices.to(_INDEX[case["index"]])
        real = _padding(case, gen)
        if real is not None:
            idx[~real] = -1
        return _State(case, logits=logits, idx=idx.contiguous(), offsets=_sequence_offsets(case, gen),
                      grad_losses=1e-3 * (1.0 + torch.rand((case["sequences"],), generator=gen, device="cuda")))
    dtype = _DTYPES[case["dtype"]]
    if family == "matvec":
        packed, scales, points = _w4(gen, 1, case["outputs"], case["inputs"], case["group"], case["zeros"], dtype)
        return _State(case, x=torch.randn((case["rows"], case["inputs"]), generator=gen, device="cuda").to(dtype),
                      weights=(packed[0], scales[0], None if points is None else points[0]))
    hidden, inter, experts = case["hidden"], case["inter"], case["experts"]
    return _State(case, x=torch.randn((case["tokens"], hidden), generator=gen, device="cuda").to(dtype), idx=_expert_routes(gen, case),
                  route_weights=torch.softmax(torch.randn((case["tokens"], case["topk"]), generator=gen, device="cuda"), dim=-1),
                  gate_up=_w4(gen, experts, 2 * inter, hidden, case["group"], case["zeros"], dtype),
                  down=_w4(gen, experts, hidden, inter, case["group"], case["zeros"], dtype))


# ---- the package's operators ---------------------------------------------------------------------------------------------------
def _router(state):
    if state.router is None:
        import deepep_amd

        c = state.case
        state.router = deepep_amd.Router(
            c["experts"], c["topk"], score=c["score"], normalize=c.get("normalize", True), scale=c.get("scale", 1.0),
            num_groups=c.get("groups", 1), num_topk_groups=c.get("topk_groups", 1), index_dtype=_INDEX[c["index"]])
    return state.router


def _run_own(state):
    case, family = state.case, state.case["family"]
    if family == "route":
        router = _router(state)
        if case["balance"]:
            idx, weights, balance = router.route_with_balance(state.logits, state.bias, state.real, sequence_offsets=state.offsets)
            grad = router.backward(state.logits, idx, topk_weights=weights, grad_weights=state.grad_weights, balance=balance,
                                   grad_losses=state.grad_losses)
            return [idx, weights, balance.losses, balance.counts, balance.tokens, grad]
        idx, weights = router.route(state.logits, state.bias, state.real)
        if not case["backward"]:
            return [idx, weights]
        return [idx, weights, router.backward(state.logits, idx, topk_weights=weights, grad_weights=state.grad_weights)]
    if family == "balance":
        router = _router(state)
        balance = router.balance_loss(state.logits, state.idx, sequence_offsets=state.offsets)
        out = [balance.losses, balance.counts, balance.tokens]
        if case["backward"]:
            out.append(router.backward(state.logits, state.idx, balance=balance, grad_losses=state.grad_losses))
        return out
    from deepep_amd import w4

    if family == "matvec":
        return [w4.matvec(state.x, w4.W4Weights(*state.weights))]
    return [w4.expert_ffn(state.x, state.idx, state.route_weights, w4.W4Weights(*state.gate_up), w4.W4Weights(*state.down))]


# ---- the same in elementary operations, 32 bits ----------------------------------------------------------------------------------
def _plain_scores(score, z):
    """Row probabilities (softmax) or the sigmoid of every logit; an expert whose logit is -inf has 0."""
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return e / e.sum(dim=1, keepdim=True).clamp_min(1e-38)


def _plain_route(case, z, bias, real):
    tokens, experts = z.shape
    scores = _plain_scores(case["score"], z)
    keys = z if case["score"] == "softmax" else scores if bias is None else scores + bias
    keys = torch.where(z == -math.inf, z, keys)
    groups = case["groups"]
    if groups > 1:
        grouped = keys.view(tokens, groups, experts // groups)
        best = torch.sort(grouped, dim=2, descending=True).values
        of_group = best[:, :, 0]
        if case["score"] == "sigmoid" and experts > groups:
            second = best[:, :, 1]
            of_group = of_group + torch.where(second == -math.inf, torch.zeros_like(second), second)
        kept = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, : case["topk_groups"]]
        allowed = torch.zeros((tokens, groups), dtype=torch.bool, device=z.device).scatter_(1, kept, True)
        keys = torch.where(allowed[:, :, None], grouped, torch.full_like(grouped, -math.inf)).view(tokens, experts)
    order = torch.sort(keys, dim=1, descending=True, stable=True)
    idx, found = order.indices[:, : case["topk"]], order.values[:, : case["topk"]] > -math.inf
    if real is not None:
        found = found & real[:, None]
    weights = torch.where(found, torch.gather(scores, 1, idx), torch.zeros((), device=z.device))
    if case["normalize"]:
        total = weights.sum(dim=1, keepdim=True)
        weights = weights / (total + 1e-20 if case["score"] == "sigmoid" else total.clamp_min(1e-38))
    return torch.where(found, idx, torch.full_like(idx, -1)).to(_INDEX[case["index"]]), weights * case["scale"], scores


def _plain_route_backward(case, scores, idx, weights, grad_weights):
    found, at = idx >= 0, idx.clamp_min(0).long()
    g = torch.where(found, grad_weights, torch.zeros_like(grad_weights)) * case["scale"]
    if case["normalize"]:
        w = weights / case["scale"]
        inner = g - (g * w).sum(dim=1, keepdim=True)
    else:
        inner = g
    chosen = torch.where(found, torch.gather(scores, 1, at), torch.zeros_like(g))
    if case["score"] == "sigmoid":
        grad = inner * chosen * (1.0 - chosen)
        if case["normalize"]:
            grad = grad / (chosen.sum(dim=1, keepdim=True) + 1e-20)
    elif case["normalize"]:
        grad = w * inner
    else:
        grad = inner * chosen
    dense = torch.zeros_like(scores).scatter_add_(1, at, torch.where(found, grad, torch.zeros_like(grad)))
    if case["score"] == "softmax" and not case["normalize"]:
        dense = dense - scores * grad.sum(dim=1, keepdim=True)
    return dense


def _plain_sequences(state, tokens):
    """[T] the sequence of each token, and their number."""
    if state.offsets is None:
        return torch.zeros((tokens,), dtype=torch.int64, device="cuda"), 1
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    return torch.searchsorted(state.offsets[1:].contiguous(), at, right=True), state.offsets.shape[0] - 1


def _plain_balance(case, state, scores, idx):
    tokens, experts = scores.shape
    of_token, sequences = _plain_sequences(state, tokens)
    p = scores if case["score"] == "softmax" else scores / (scores.sum(dim=1, keepdim=True) + 1e-20)
    real = (idx >= 0).any(dim=1)
    member = torch.zeros((sequences, tokens), device="cuda").scatter_(0, of_token[None, :], real[None, :].to(torch.float32))
    cell = torch.where(idx >= 0, of_token[:, None] * experts + idx, torch.full_like(idx, sequences * experts)).reshape(-1).long()
    counts = torch.zeros((sequences * experts + 1,), dtype=torch.int32, device="cuda").scatter_add_(0, cell, torch.ones_like(cell, dtype=torch.int32))
    counts = counts[:-1].view(sequences, experts)
    held = member.sum(dim=1)
    mean = (member @ p) / held.clamp_min(1.0)[:, None]
    load = counts.to(torch.float32) * experts / counts.sum(dim=1, keepdim=True).clamp_min(1)
    return p, real, of_token, load, held, (load * mean).sum(dim=1), counts, held.to(torch.int32)


def _plain_balance_backward(case, state, scores, p, real, of_token, load, held):
    a = torch.where(real, (state.grad_losses / held.clamp_min(1.0))[of_token], torch.zeros((), device="cuda"))[:, None]
    f = load[of_token]
    inner = f - (f * p).sum(dim=1, keepdim=True)
    if case["score"] == "softmax":
        return a * p * inner
    return a * inner * scores * (1.0 - scores) / (scores.sum(dim=1, keepdim=True) + 1e-20)


def _plain_weights(packed, scales, points, group):
    """The matrices' values in 32 bits, [..., N, K]."""
    q = torch.stack([packed & 15, packed >> 4], dim=-1).view(*packed.shape[:-1], -1, group).to(torch.float32)
    q -= 8.0 if points is None else points.to(torch.float32)[..., None]
    q *= scales.to(torch.float32)[..., None]
    return q.view(*packed.shape[:-1], -1)


def _plain_product(weights, at, group, x):
    """[R, N]: row r's vector times the matrix of expert at[r]."""
    packed, scales, points = weights
    w = _plain_weights(packed[at], scales[at], None if points is None else points[at], group)
    return (w @ x[:, :, None])[:, :, 0]


def _run_plain(state):
    case, family = state.case, state.case["family"]
    if family == "route":
        idx, weights, scores = _plain_route(case, state.logits.to(torch.float32), state.bias, state.real)
        if not case["backward"]:
            return [idx, weights]
        grad = _plain_route_backward(case, scores, idx, weights, state.grad_weights)
        if not case["balance"]:
            return [idx, weights, grad.to(state.logits.dtype)]
        p, real, of_token, load, held, losses, counts, members = _plain_balance(case, state, scores, idx)
        grad = grad + _plain_balance_backward(case, state, scores, p, real, of_token, load, held)
        return [idx, weights, losses, counts, members, grad.to(state.logits.dtype)]
    if family == "balance":
        scores = _plain_scores(case["score"], state.logits.to(torch.float32))
        p, real, of_token, load, held, losses, counts, members = _plain_balance(case, state, scores, state.idx)
        if not case["backward"]:
            return [losses, counts, members]
        grad = _plain_balance_backward(case, state, scores, p, real, of_token, load, held)
        return [losses, counts, members, grad.to(state.logits.dtype)]
    if family == "matvec":
        w = _plain_weights(*state.weights, case["group"])
        return [(state.x.to(torch.float32) @ w.t()).to(state.x.dtype)]
    tokens, topk = state.idx.shape
    at = state.idx.clamp_min(0).view(-1)
    routed = torch.where(state.idx >= 0, state.route_weights, torch.zeros_like(state.route_weights))
    x = state.x.to(torch.float32)[:, None, :].expand(tokens, topk, -1).reshape(tokens * topk, -1)
    gate, up = _plain_product(state.gate_up, at, case["group"], x).chunk(2, dim=1)
    h = gate / (1.0 + torch.exp(-gate)) * up
    y = _plain_product(state.down, at, case["group"], h).view(tokens, topk, -1)
    return [(y * routed[:, :, None]).sum(dim=1).to(state.x.dtype)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------
def _exact_choice(case, z, bias, real):
    """Expert ids [T,K], -1 where nothing is left, by repeated search for the best remaining key.  Keys are 32-bit values by
    definition, so each score is rounded to 32 bits here, once."""
    tokens, experts = z.shape
    keys = z.float() if case["score"] == "softmax" else torch.sigmoid(z).float() + (0.0 if bias is None else bias)
    keys[torch.isneginf(z)] = -math.inf
    if real is not None:
        keys[~real] = -math.inf
    if case["groups"] > 1:
        width = experts // case["groups"]
        blocks = keys.split(width, dim=1)
        if case["score"] == "softmax":
            value = torch.stack([b.max(dim=1).values for b in blocks], dim=1)
        else:
            best = [b.topk(min(2, width), dim=1).values for b in blocks]
            value = torch.stack([b[:, 0] + b[:, 1:].masked_fill(b[:, 1:].isneginf(), 0.0).sum(dim=1) for b in best], dim=1)
        allowed = torch.zeros_like(value, dtype=torch.bool)
        for _ in range(case["topk_groups"]):
            pick = value.masked_fill(allowed, -math.inf)
            first = (pick == pick.max(dim=1, keepdim=True).values).logical_and(~allowed).to(torch.int8).argmax(dim=1, keepdim=True)
            allowed.scatter_(1, first, True)
        keys = keys.masked_fill(~allowed.repeat_interleave(width, dim=1), -math.inf)
    chosen = []
    for _ in range(case["topk"]):
        best = keys.max(dim=1, keepdim=True).values
        first = (keys == best).to(torch.int8).argmax(dim=1, keepdim=True)
        chosen.append(torch.where(best > -math.inf, first, torch.full_like(first, -1)))
        keys = keys.scatter(1, first, -math.inf)
    return torch.cat(chosen, dim=1)


def _exact_weights(case, z, idx):
    """Route weights as a function of the logits that autograd can follow."""
    picked = torch.gather(z, 1, idx.clamp_min(0)).masked_fill(idx < 0, -math.inf)
    if case["score"] == "sigmoid":
        w = torch.sigmoid(picked)
        return case["scale"] * (w / (w.sum(dim=1, keepdim=True) + 1e-20) if case["normalize"] else w)
    norm = torch.logsumexp(picked if case["normalize"] else z, dim=1, keepdim=True)
    return case["scale"] * torch.exp(picked - norm.masked_fill(norm.isneginf(), 0.0))


def _exact_losses(case, z, idx, offsets):
    """The sequences' balance losses, counts and token numbers; the losses as a function that autograd can follow."""
    tokens, experts = z.shape
    if case["score"] == "softmax":
        norm = torch.logsumexp(z, dim=1, keepdim=True)
        p = torch.exp(z - norm.masked_fill(norm.isneginf(), 0.0))
    else:
        s = torch.sigmoid(z)
        p = s / (s.sum(dim=1, keepdim=True) + 1e-20)
    bounds = [0, tokens] if offsets is None else offsets.tolist()
    losses, counts, members = [], [], []
    for begin, end in zip(bounds[:-1], bounds[1:]):
        routes = idx[begin:end]
        held = (routes >= 0).any(dim=1)
        count = torch.bincount(routes[routes >= 0].reshape(-1).long(), minlength=experts)
        number = int(held.sum())
        losses.append((p[begin:end][held].sum(dim=0) / max(1, number) * count.double() * experts / max(1, int(count.sum()))).sum())
        counts.append(count.to(torch.int32))
        members.append(number)
    return torch.stack(losses), torch.stack(counts), torch.tensor(members, dtype=torch.int32, device=z.device)


def _exact_matrix(packed, scales, points, group):
    low, high = (packed % 16).double(), (packed // 16).double()
    q = torch.empty((*packed.shape[:-1], packed.shape[-1] * 2), dtype=torch.float64, device=packed.device)
    q[..., 0::2], q[..., 1::2] = low, high
    shift = torch.full_like(scales, 8.0, dtype=torch.float64) if points is None else points.double()
    return (q - shift.repeat_interleave(group, dim=-1)) * scales.double().repeat_interleave(group, dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    family = case["family"]
    if family in ("route", "balance"):
        z = state.logits.double().requires_grad_(case["backward"])
        if family == "balance":
            losses, counts, members = _exact_losses(case, z, state.idx, state.offsets)
            out = [losses.detach(), counts, members]
            total = (losses * state.grad_losses.double()).sum()
        else:
            idx = _exact_choice(case, z.detach(), state.bias, state.real)
            weights = _exact_weights(case, z, idx)
            out = [None, weights.detach()]  # (two keys a rounding apart may change places)
            if not case["backward"]:
                return out
            total = (weights * state.grad_weights.double()).sum()
            if case["balance"]:
                losses, counts, members = _exact_losses(case, z, idx, state.offsets)
                out += [losses.detach(), None, members]
                total = total + (losses * state.grad_losses.double()).sum()
        if case["backward"]:
            total.backward()
            out.append(torch.nan_to_num(z.grad))
        return out
    if family == "matvec":
        return [state.x.double() @ _exact_matrix(*state.weights, case["group"]).t()]
    y = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")

    def matrix(weights, e):
        return _exact_matrix(weights[0][e], weights[1][e], None if weights[2] is None else weights[2][e], case["group"])

    for e in sorted(set(state.idx[state.idx >= 0].tolist())):
        token, slot = (state.idx == e).nonzero(as_tuple=True)
        both = state.x[token].double() @ matrix(state.gate_up, e).t()
        gate, up = both[:, : case["inter"]], both[:, case["inter"]:]
        out = (torch.sigmoid(gate) * gate * up) @ matrix(state.down, e).t()
        y.index_add_(0, token, out * state.route_weights[token, slot].double()[:, None])
    return [y]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once (expected values of the routing)."""
    family = case["family"]
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if family in ("route", "balance"):
        cells, routes = case["tokens"] * case["experts"], case["tokens"] * case["topk"]
        index = {"int64": 8, "int32": 4}[case["index"]]
        total = cells * size + routes * index + (case["tokens"] if case["padding"] else 0)
        flops = 4 * cells
        balance = family == "balance" or case["balance"]
        if family == "route":
            total += routes * 4 + (case["experts"] * 4 if case["bias"] else 0)
        if balance:
            total += case["sequences"] * (case["experts"] + 3) * 4
            flops += 2 * cells
        if case["backward"]:
            total += cells * size + (routes * 4 if family == "route" else 0)
            flops += 6 * cells if balance or (case["score"] == "softmax" and not case["normalize"]) else 8 * routes
        return {"bytes": total, "flops": flops}
    per_weight = 0.5 + (size + (1 if case["zeros"] else 0)) / case["group"]
    if family == "matvec":
        rows, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": n * k * per_weight + rows * (k + n) * size, "flops": 2 * rows * n * k}
    served = case["tokens"] * case["topk"] - int(case["masked"] * case["tokens"] * case["topk"])
    popularity = [(e + 1.0) ** -case["skew"] for e in range(case["experts"])]
    each = served / sum(popularity)
    touched = sum(1.0 - (1.0 - min(1.0, each * p / case["tokens"])) ** case["tokens"] for p in popularity)
    weights = 3 * case["inter"] * case["hidden"]
    return {"bytes": touched * weights * per_weight + case["tokens"] * case["hidden"] * 2 * size + case["tokens"] * case["topk"] * 12,
            "flops": 2 * served * weights}
