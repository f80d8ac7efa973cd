"""Router, balance loss and their gradients on the GPU against the 64-bit oracle.

Expert ids and counts have to be equal.  Logits lie on a grid (1/16) so that equal keys are equal bits on both sides, and rows with
two keys or group scores closer than 2e-6 without being equal are drawn again: the order is then the same in 32 and in 64 bits.
Weights: exp is off by an ulp, its argument by |z - max| 2^-24 (logits up to 6: 12 ulp), a sum of up to 1024 terms in a tree by ten
more, divide and scale by one each: 32 * 2^-24 = 2e-6 of the value, 4e-6 here.  Gradients are differences of such terms, so their
bound is relative to the largest of a token; a narrower logits type adds half its last place."""

import numpy as np
import pytest
import torch

from oracle import router as orouter

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
PLACE = {"fp32": 2.0**-23, "bf16": 2.0**-8, "fp16": 2.0**-10}
NEAR = 2e-6


def _close_calls(z, score, bias, groups):
    """Which rows hold two different keys, or group scores, nearer than NEAR."""
    keys = z if score == "softmax" else orouter.sigmoid(z) + (0.0 if bias is None else bias)
    keys = np.where(np.isneginf(z), -np.inf, keys)
    found = np.zeros(len(z), dtype=bool)
    values = [keys]
    if groups > 1:
        best = -np.sort(-keys.reshape(len(z), groups, -1), axis=2)
        both = best[:, :, 0]
        if score == "sigmoid" and best.shape[2] > 1:
            both = both + np.where(np.isneginf(best[:, :, 1]), 0.0, best[:, :, 1])
        values.append(both)
    for value in values:
        order = np.sort(np.where(np.isneginf(value), -1e9, value), axis=1)
        gap = np.diff(order, axis=1)
        found |= ((gap > 0) & (gap < NEAR)).any(axis=1)
    return found


def _logits(rng, tokens, experts, score, bias, groups, closed):
    def draw(n):
        z = rng.integers(-96, 97, size=(n, experts)) / 16.0
        z[rng.random((n, experts)) < closed] = -np.inf
        return z

    z = draw(tokens)
    for _ in range(50):
        again = _close_calls(z, score, bias, groups)
        if not again.any():
            break
        z[again] = draw(int(again.sum()))
    return z


# tokens, experts, topk, score, normalize, scale, groups, topk_groups, bias, dtype, index, masked, closed
CASES = [
    (1, 1, 1, "softmax", True, 1.0, 1, 1, False, "fp32", torch.int64, 0.0, 0.0),
    (1, 256, 8, "sigmoid", True, 2.5, 8, 4, True, "fp32", torch.int64, 0.0, 0.0),
    (7, 65, 5, "softmax", False, 1.0, 1, 1, False, "bf16", torch.int32, 0.2, 0.05),
    (33, 160, 6, "softmax", True, 1.0, 8, 3, False, "fp32", torch.int64, 0.2, 0.0),
    (130, 176, 10, "sigmoid", False, 0.5, 8, 5, True, "bf16", torch.int32, 0.1, 0.1),
    (64, 1024, 32, "sigmoid", True, 1.0, 16, 7, True, "fp32", torch.int64, 0.0, 0.0),
    (65, 1000, 32, "softmax", False, 3.0, 1, 1, False, "fp16", torch.int64, 0.0, 0.02),
    (129, 384, 6, "softmax", True, 1.0, 1, 1, False, "bf16", torch.int32, 0.0, 0.0),
    (50, 12, 4, "sigmoid", True, 1.0, 4, 2, False, "fp16", torch.int64, 0.0, 0.3),
    (50, 12, 4, "softmax", True, 1.0, 12, 4, False, "fp32", torch.int64, 0.0, 0.5),
    (40, 8, 8, "sigmoid", True, 1.0, 8, 8, True, "fp32", torch.int64, 0.0, 0.6),
    (301, 512, 1, "sigmoid", True, 1.0, 2, 1, True, "fp32", torch.int64, 0.05, 0.0),
    (90, 255, 3, "sigmoid", False, 1.0, 3, 2, False, "fp32", torch.int32, 0.0, 0.0),
    (21, 129, 9, "softmax", True, -1.5, 1, 1, False, "bf16", torch.int64, 0.0, 0.9),
]


def _case(number):
    tokens, experts, topk, score, normalize, scale, groups, topk_groups, biased, dtype, index, masked, closed = CASES[number]
    from deepep_amd import Router

    rng = np.random.default_rng(100 + number)
    bias = rng.integers(-8, 9, size=experts) / 8.0 if biased else None
    z = _logits(rng, tokens, experts, score, bias, groups, closed)
    real = rng.random(tokens) >= masked if masked else None
    router = Router(experts, topk, score=score, normalize=normalize, scale=scale, num_groups=groups, num_topk_groups=topk_groups, index_dtype=index)
    logits = torch.from_numpy(z).to(DTYPES[dtype]).cuda()
    assert np.array_equal(logits.double().cpu().numpy(), z)  # the grid is exact in every type
    return router, rng, z, logits, bias, real


def _route(router, logits, bias, real):
    return router.route(logits, None if bias is None else torch.from_numpy(bias).float().cuda(), None if real is None else torch.from_numpy(real).cuda())


def _oracle_ids(router, z, bias, real):
    return [orouter.choose(z[t], router.num_topk, router.score, bias, real is None or real[t], router.num_groups, router.num_topk_groups)
            for t in range(len(z))]


@pytest.mark.parametrize("number", range(len(CASES)))
def test_route(number):
    router, rng, z, logits, bias, real = _case(number)
    idx, weights = _route(router, logits, bias, real)
    assert idx.dtype == router.index_dtype
    ids = _oracle_ids(router, z, bias, real)
    np.testing.assert_array_equal(idx.cpu().numpy(), np.array(ids))
    want = np.stack([orouter.weights_of(z[t], ids[t], router.score, router.normalize, router.scale) for t in range(len(z))])
    np.testing.assert_allclose(weights.double().cpu().numpy(), want, rtol=4e-6, atol=1e-30)
    again = _route(router, logits, bias, real)
    assert torch.equal(idx, again[0]) and torch.equal(weights.view(torch.int32), again[1].view(torch.int32))


def _offsets(rng, tokens, sequences):
    return None if sequences == 1 else np.array([0, *sorted(rng.integers(0, tokens + 1, size=sequences - 1)), tokens])


def _check_gradient(got, want, terms, dtype):
    """terms: [T,1] what a token's gradient is a difference of."""
    bound = 1e-5 * terms + PLACE[dtype] * np.abs(want) + (6e-8 if dtype == "fp16" else 1e-37)
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("number", range(len(CASES)))
@pytest.mark.parametrize("sequences", [1, 5])
def test_gradients(number, sequences):
    router, rng, z, logits, bias, real = _case(number)
    dtype, tokens = CASES[number][9], len(z)
    idx, weights = _route(router, logits, bias, real)
    ids = idx.cpu().numpy()
    offsets = _offsets(rng, tokens, sequences)
    device_offsets = None if offsets is None else torch.from_numpy(offsets).int().cuda()
    balance = router.balance_loss(logits, idx, device_offsets)
    losses, counts, members = orouter.balance(z, ids, router.score, offsets)
    np.testing.assert_array_equal(balance.counts.cpu().numpy(), counts)
    np.testing.assert_array_equal(balance.tokens.cpu().numpy(), members)
    np.testing.assert_allclose(balance.losses.double().cpu().numpy(), losses, rtol=2e-5, atol=0)
    g = rng.normal(size=ids.shape).astype(np.float32)
    g_losses = rng.normal(size=len(losses)).astype(np.float32)
    through = np.stack([orouter.weights_gradient(z[t], ids[t], g[t], router.score, router.normalize, router.scale) for t in range(tokens)])
    from_balance = orouter.balance_gradient(z, ids, g_losses, router.score, offsets)
    terms = np.abs(g).max(axis=1, keepdims=True) * abs(router.scale)
    load = np.abs(counts * z.shape[1] / np.maximum(counts.sum(axis=1, keepdims=True), 1)).max(axis=1) * np.abs(g_losses) / np.maximum(members, 1)
    of_token = np.zeros(tokens, dtype=int) if offsets is None else np.searchsorted(offsets[1:], np.arange(tokens), side="right")
    balance_terms = load[of_token][:, None]
    device_g, device_g_losses = torch.from_numpy(g).cuda(), torch.from_numpy(g_losses).cuda()
    got = router.backward(logits, idx, topk_weights=weights, grad_weights=device_g)
    assert got.dtype == logits.dtype
    _check_gradient(got, through, terms, dtype)
    _check_gradient(router.backward(logits, idx, balance=balance, grad_losses=device_g_losses), from_balance, balance_terms, dtype)
    both = router.backward(logits, idx, topk_weights=weights, grad_weights=device_g, balance=balance, grad_losses=device_g_losses)
    _check_gradient(both, through + from_balance, terms + balance_terms, dtype)
    offsets_of_both = dict(sequence_offsets=device_offsets)
    idx2, weights2, balance2 = router.route_with_balance(
        logits, None if bias is None else torch.from_numpy(bias).float().cuda(), None if real is None else torch.from_numpy(real).cuda(), **offsets_of_both)
    assert torch.equal(idx2, idx) and torch.equal(weights2.view(torch.int32), weights.view(torch.int32))
    assert torch.equal(balance2.counts, balance.counts) and torch.equal(balance2.tokens, balance.tokens)
    np.testing.assert_allclose(balance2.losses.double().cpu().numpy(), losses, rtol=2e-5, atol=0)


@pytest.mark.parametrize("tokens,experts,topk,sequences", [(5000, 64, 4, 1), (5000, 256, 8, 40), (1, 16, 2, 3), (3000, 160, 6, 3000)])
def test_balance_of_many_tokens(tokens, experts, topk, sequences):
    """Chunks that hold many sequences, sequences that span many chunks, empty ones; ids of either width, some outside the range."""
    from deepep_amd import Router

    rng = np.random.default_rng(tokens + sequences)
    z = rng.normal(size=(tokens, experts)).astype(np.float32)
    ids = np.argsort(rng.random((tokens, experts)), axis=1)[:, :topk]
    ids[rng.random(tokens) < 0.1] = -1
    ids[rng.random(ids.shape) < 0.05] = experts + 3
    offsets = _offsets(rng, tokens, sequences)
    losses, counts, members = orouter.balance(z, np.where(ids < experts, ids, -1), "softmax", offsets)
    for index in (torch.int64, torch.int32):
        balance = Router(experts, topk).balance_loss(torch.from_numpy(z).cuda(), torch.from_numpy(ids).to(index).cuda(),
                                                     None if offsets is None else torch.from_numpy(offsets).int().cuda())
        np.testing.assert_array_equal(balance.counts.cpu().numpy(), counts)
        np.testing.assert_array_equal(balance.tokens.cpu().numpy(), members)
        np.testing.assert_allclose(balance.losses.double().cpu().numpy(), losses, rtol=2e-5, atol=0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinities_and_nans(score):
    """A NaN is chosen first and shows in the weights; +inf is chosen; -inf never; a row of -inf has no route and no gradient."""
    from deepep_amd import Router

    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[0.0, nan, 1.0, 2.0], [0.0, inf, 1.0, 2.0], [-inf, -inf, -inf, -inf], [-inf, 3.0, -inf, -inf], [-inf, nan, -inf, 1.0],
                      [-3e38, -3e38, -3.4028234663852886e38, 0.0]]).cuda()
    router = Router(4, 2, score=score)
    idx, weights = router.route(z)
    assert idx.tolist() == [[1, 3], [1, 3], [-1, -1], [1, -1], [1, 3], [3, 0]]
    weights = weights.cpu()
    assert torch.isnan(weights[0]).all() and torch.isnan(weights[4]).all()
    assert weights[2].tolist() == [0, 0] and weights[3].tolist() == [1, 0] and weights[5].tolist() == [1, 0]
    grad = router.backward(z, idx, topk_weights=weights.cuda(), grad_weights=torch.ones(6, 2).cuda()).cpu()
    assert grad[2].tolist() == [0] * 4 and grad[3].tolist() == [0] * 4 and torch.isfinite(grad[5]).all()
    finite = z[[2, 3, 5]].contiguous()
    idx = idx[[2, 3, 5]].contiguous()
    balance = router.balance_loss(finite, idx)
    assert balance.tokens.tolist() == [2] and torch.isfinite(balance.losses).all()
    grad = router.backward(finite, idx, balance=balance, grad_losses=torch.ones(1).cuda())
    assert torch.isfinite(grad).all() and grad[0].tolist() == [0] * 4


@pytest.mark.parametrize("experts,groups,topk_groups", [
    (64, 4, 2), (64, 16, 5), (64, 64, 9), (63, 7, 3), (128, 8, 4), (128, 32, 8), (256, 8, 4), (256, 4, 3), (256, 64, 31), (240, 6, 2), (512, 4, 1),
    (512, 8, 7), (1024, 64, 20), (1024, 2, 1),
])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_with_ties(experts, groups, topk_groups, score):
    """Groups of one lane to all of them, whole registers or not, with equal scores everywhere: the lower group and expert come first.  Softmax: small
    whole logits; sigmoid: logits of zero, whose score is 1/2 exactly, and biases of eighths, so that sums are exact."""
    from deepep_amd import Router

    rng = np.random.default_rng(experts + groups)
    tokens, bias = 40, None
    z = rng.integers(-2, 3, size=(tokens, experts)).astype(np.float64)
    if score == "sigmoid":
        z, bias = np.zeros((tokens, experts)), rng.integers(-2, 3, size=experts) / 8.0
    z[rng.random(z.shape) < 0.4] = -np.inf
    z[5, : experts - experts // groups] = -np.inf  # only the last group has any
    topk = min(8, experts // groups * topk_groups)
    router = Router(experts, topk, score=score, num_groups=groups, num_topk_groups=topk_groups)
    idx, _ = router.route(torch.from_numpy(z).float().cuda(), None if bias is None else torch.from_numpy(bias).float().cuda())
    np.testing.assert_array_equal(idx.cpu().numpy(), _oracle_ids(router, z, bias, None))


def test_underflowing_scores():
    """Sigmoids that are all zero in fp32: the weights and gradients stay finite, ties go to the lowest index."""
    from deepep_amd import Router

    z = torch.full((3, 8), -200.0).cuda()
    router = Router(8, 3, score="sigmoid")
    idx, weights, balance = router.route_with_balance(z)
    assert idx.tolist() == [[0, 1, 2]] * 3 and not weights.any() and balance.losses.tolist() == [0.0]
    grad = router.backward(z, idx, topk_weights=weights, grad_weights=torch.ones(3, 3).cuda(), balance=balance, grad_losses=torch.ones(1).cuda())
    assert torch.isfinite(grad).all()


def test_empty_batch():
    from deepep_amd import Router

    router = Router(16, 4)
    z = torch.empty((0, 16)).cuda()
    idx, weights, balance = router.route_with_balance(z, sequence_offsets=torch.zeros(4, dtype=torch.int32).cuda())
    assert idx.shape == weights.shape == (0, 4)
    assert balance.losses.tolist() == [0.0] * 3 and balance.tokens.tolist() == [0] * 3 and not balance.counts.any()
    grad = router.backward(z, idx, topk_weights=weights, grad_weights=torch.empty((0, 4)).cuda(), balance=balance, grad_losses=torch.ones(3).cuda())
    assert grad.shape == (0, 16)


def _device_step(router, logits, bias, offsets, g, g_losses):
    idx, weights, balance = router.route_with_balance(logits, bias, sequence_offsets=offsets)
    grad = router.backward(logits, idx, topk_weights=weights, grad_weights=g, balance=balance, grad_losses=g_losses)
    return [idx, weights, balance.losses, balance.counts, balance.tokens, grad]


def test_other_streams_and_odd_addresses():
    """Inputs made on another stream, views whose first element is at an odd place: the same bits."""
    from deepep_amd import Router

    gen = torch.Generator(device="cuda").manual_seed(3)
    router = Router(96, 6, score="sigmoid", num_groups=4, num_topk_groups=2)
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.randn((500, 96), generator=gen, device="cuda").to(dtype)
        bias = torch.randn((96,), generator=gen, device="cuda")
        offsets = torch.tensor([0, 100, 100, 500], dtype=torch.int32).cuda()
        g, g_losses = torch.randn((500, 6), generator=gen, device="cuda"), torch.randn((3,), generator=gen, device="cuda")
        want = _device_step(router, logits, bias, offsets, g, g_losses)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            shifted = torch.empty(500 * 96 + 1, dtype=dtype, device="cuda")[1:].view(500, 96)
            shifted.copy_(logits)
            odd_bias = torch.empty(97, device="cuda")[1:]
            odd_bias.copy_(bias)
            got = _device_step(router, shifted, odd_bias, offsets, g, g_losses)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_graph_replays():
    from deepep_amd import Router

    gen = torch.Generator(device="cuda").manual_seed(4)
    router = Router(160, 6, score="sigmoid", num_groups=8, num_topk_groups=3)
    logits = torch.randn((3000, 160), generator=gen, device="cuda")
    bias = torch.randn((160,), generator=gen, device="cuda")
    offsets = torch.tensor([0, 1, 1500, 3000], dtype=torch.int32).cuda()
    g, g_losses = torch.randn((3000, 6), generator=gen, device="cuda"), torch.ones((3,), device="cuda")
    _device_step(router, logits, bias, offsets, g, g_losses)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        captured = _device_step(router, logits, bias, offsets, g, g_losses)
    for _ in range(4):
        logits.copy_(torch.randn((3000, 160), generator=gen, device="cuda"))
        g.copy_(torch.randn((3000, 6), generator=gen, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, _device_step(router, logits, bias, offsets, g, g_losses)):
            assert torch.equal(a, b)


def test_refusals():
    from deepep_amd import Router

    router = Router(16, 4)
    z = torch.zeros((8, 16)).cuda()
    idx, weights = router.route(z)
    bad = [
        lambda: router.route(z.cpu()),
        lambda: router.route(z.double()),
        lambda: router.route(z[:, :8]),
        lambda: router.route(z.t().contiguous().t()),
        lambda: router.route(z, bias=torch.zeros(16).cuda()),
        lambda: Router(16, 4, score="sigmoid").route(z, bias=torch.zeros(15).cuda()),
        lambda: router.route(z, token_mask=torch.ones(8, dtype=torch.uint8).cuda()),
        lambda: router.route(z, token_mask=torch.ones(7, dtype=torch.bool).cuda()),
        lambda: router.balance_loss(z, idx[:, :3].contiguous()),
        lambda: router.balance_loss(z, idx.float()),
        lambda: router.balance_loss(z, idx, torch.tensor([0, 8]).cuda()),
        lambda: router.balance_loss(z, idx, torch.tensor([0], dtype=torch.int32).cuda()),
        lambda: router.backward(z, idx),
        lambda: router.backward(z, idx, grad_weights=weights),
        lambda: router.backward(z, idx, topk_weights=weights, grad_weights=weights[:4]),
        lambda: router.backward(z, idx, balance=router.balance_loss(z, idx)),
        lambda: router.backward(z, idx, balance=router.balance_loss(z, idx), grad_losses=torch.ones(2).cuda()),
        lambda: router.backward(z[:4].contiguous(), idx, topk_weights=weights, grad_weights=weights),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_native_and_python_layers_agree():
    """Logits that carry a gradient go through the Python layer; the bits are the same."""
    from deepep_amd import Router

    gen = torch.Generator(device="cuda").manual_seed(9)
    for score, index in (("sigmoid", torch.int64), ("softmax", torch.int32)):
        router = Router(48, 5, score=score, normalize=score == "sigmoid", num_groups=6, num_topk_groups=3, index_dtype=index)
        logits = torch.randn((300, 48), generator=gen, device="cuda")
        bias = torch.randn((48,), generator=gen, device="cuda") if score == "sigmoid" else None
        mask = torch.rand((300,), generator=gen, device="cuda") < 0.8
        offsets = torch.tensor([0, 77, 300], dtype=torch.int32).cuda()
        g, g_losses = torch.randn((300, 5), generator=gen, device="cuda"), torch.randn((2,), generator=gen, device="cuda")

        def step(logits):
            idx, weights = router.route(logits, bias, mask)
            idx2, weights2, balance = router.route_with_balance(logits, bias, mask, sequence_offsets=offsets)
            again = router.balance_loss(logits, idx, offsets)
            grad = router.backward(logits, idx, topk_weights=weights, grad_weights=g, balance=balance, grad_losses=g_losses)
            return [idx, weights, idx2, weights2, *balance[:3], *again[:3], grad]

        native = step(logits)
        assert router._native.route(logits, bias, mask) is not None
        leaf = logits.clone().requires_grad_()
        assert router._native.route(leaf, bias, mask) is None
        for a, b in zip(native, step(leaf)):
            assert torch.equal(a, b.detach())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,groups", [(4, 1), (300, 1), (256, 4)])
def test_slots_without_a_route_weigh_nothing(score, normalize, experts, groups):
    """Padding rows may hold anything, and a row that runs out of experts may hold a NaN or +inf among those it has: the slots that are left
    get -1 and 0, and padding takes no part in loss or gradient."""
    from deepep_amd import Router

    inf, nan = float("inf"), float("nan")
    gen = torch.Generator().manual_seed(experts)
    z = torch.randn(10, experts, generator=gen)
    real = torch.tensor([True, False, False, False, True, True, True, False, True, True])
    z[1], z[2, 1], z[3, 2], z[7] = nan, nan, inf, -inf
    z[1, 0] = 0.0
    for row, first in ((4, nan), (5, inf), (6, 1.0)):
        z[row] = -inf
        z[row, 3] = first
    router = Router(experts, 3, score=score, normalize=normalize, scale=-1.5, num_groups=groups, num_topk_groups=min(groups, 2))
    z, real_gpu = z.cuda(), real.cuda()
    idx, weights = router.route(z, token_mask=real_gpu)
    idx2, weights2, balance = router.route_with_balance(z, token_mask=real_gpu)
    assert torch.equal(idx, idx2) and torch.equal(weights.view(torch.int32), weights2.view(torch.int32))
    assert (idx[~real_gpu] == -1).all() and (idx[4:7] == torch.tensor([3, -1, -1]).cuda()).all() and (idx[[0, 8, 9]] >= 0).all()
    assert (weights[idx < 0] == 0).all(), weights.tolist()
    assert torch.isnan(weights[4, 0]) and torch.isfinite(weights[[0, 6, 8, 9]]).all()
    kept = torch.tensor([0, 1, 2, 3, 6, 7, 8, 9]).cuda()
    z, idx, weights, real = z[kept].contiguous(), idx[kept].contiguous(), weights[kept].contiguous(), real[kept.cpu()]
    again = router.balance_loss(z, idx)
    assert again.tokens.tolist() == [int(real.sum())] and torch.isfinite(again.losses).all()
    grad = router.backward(z, idx, topk_weights=weights, grad_weights=torch.full_like(weights, nan).masked_fill(idx >= 0, 1.0), balance=again,
                           grad_losses=torch.ones(1).cuda())
    assert torch.isfinite(grad).all() and not grad[~real.cuda()].any()


def test_sigmoid_keys_have_the_bits_of_a_divide():
    """Every float from 2^-25 to 128 in magnitude as a logit (below, the sum is 2): the scores are 1 / (1 + torch.exp(-z)) bit for bit, on both sides of where the sum leaves
    the reciprocal's range (-86) and where the sigmoid becomes subnormal and zero, and ids and biased ids are in the order of such keys."""
    from deepep_amd import Router

    experts = 32
    bias = torch.linspace(-0.5, 0.5, experts, device="cuda")[torch.randperm(experts, generator=torch.Generator().manual_seed(1)).cuda()]
    router = Router(experts, experts, score="sigmoid", normalize=False)
    for sign in (0, 1 << 31):
        for exponent in range(102, 134):  # of 2^-25 to 2^6
            bits = torch.arange(1 << 23, dtype=torch.int64, device="cuda") + (exponent << 23) + sign
            z = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32)
            z = z.view(experts, -1).t().contiguous()  # (a row's logits are spread over the binade)
            want = 1.0 / (1.0 + torch.exp(-z))
            for keys, given in ((want, None), (want + bias, bias)):
                idx, weights = router.route(z, given)
                assert torch.equal(idx, torch.sort(keys, dim=1, descending=True, stable=True).indices), (sign, exponent)
                assert torch.equal(weights.view(torch.int32), want.gather(1, idx).view(torch.int32)), (sign, exponent)
