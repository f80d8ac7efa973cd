"""The norm, the feed-forward block and the 8-bit products as a layer uses them, next to the router, the exchange and the other experts: a whole block's training step
against 64-bit autograd, its serving form against the dequantised weights, and the norm's 8-bit outputs where the framework takes them."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, INTER, EXPERTS, TOPK = 120, 256, 128, 16, 3


@pytest.fixture
def block():
    from examples.routed_layer import Block, RoutedLayer

    layer = RoutedLayer(HIDDEN, INTER, EXPERTS, TOPK, max_tokens=TOKENS, scale=2.5, seed=5)
    made = Block(layer)
    made.norm += torch.randn(HIDDEN, generator=torch.Generator().manual_seed(1)).cuda() / 4
    yield made
    layer.destroy()


def _rows(seed, count=TOKENS):
    return torch.randn(count, HIDDEN, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _near(got, want, bound, what):
    got, want = got.double().cpu(), want.double().cpu()
    err = ((got - want).norm() / want.norm()).item()
    assert err <= bound, (what, err)


def _exact(block, stream, topk_idx, parameters):
    """The block in 64 bits on the stored stream, with the choice of experts that was made."""
    norm, shared_gate_up, shared_down, gate, gate_up, down = parameters
    normed = stream * (stream.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * norm
    picked = torch.sigmoid(normed @ gate.T).gather(1, topk_idx)
    weights = 2.5 * picked / picked.sum(dim=1, keepdim=True)
    out = torch.zeros_like(stream)
    for e in range(EXPERTS):
        for s in range(TOPK):
            chosen = (topk_idx[:, s] == e).nonzero()[:, 0]
            g, u = (normed[chosen] @ gate_up[e].T).chunk(2, dim=1)
            out = out.index_add(0, chosen, weights[chosen, s, None] * ((F.silu(g) * u) @ down[e].T))
    g, u = (normed @ shared_gate_up.T).chunk(2, dim=1)
    return out + (F.silu(g) * u) @ shared_down.T


def test_training_step(block):
    """Up to ten roundings to BF16 follow one another (norm, rows, h, both outputs, their sum; and back): each off by 2^-8 / sqrt(3) in the mean, together 0.007."""
    x, residual, grad_out, grad_stream = (_rows(seed) for seed in (2, 3, 4, 5))
    out, stream, _, saved = block.forward(x.cuda(), residual.cuda())
    assert torch.equal(stream.cpu(), (x.float() + residual.float()).bfloat16())
    grads = block.backward(grad_out.cuda(), grad_stream.cuda(), saved)
    layer = block.layer
    leaves = [t.double().cpu().requires_grad_(True) for t in (stream, block.norm, block.shared_gate_up, block.shared_down, layer.gate, layer.gate_up, layer.down)]
    want = _exact(block, leaves[0], saved[1][2].cpu(), leaves[1:])
    _near(out, want.detach(), 1e-2, "out")
    ((want * grad_out.double()).sum() + (leaves[0] * grad_stream.double()).sum()).backward()
    for grad, leaf, name in zip(grads, leaves, ("x", "norm", "shared gate_up", "shared down", "gate", "gate_up", "down")):
        _near(grad, leaf.grad, 1e-2, name)


@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_decode(block, tokens):
    """Against the dequantised weights: what is left is the tokens in 8 bits, twice.  A code is off by 1/2 of a step of max/127 at most, in the mean by 1 / sqrt(12) of
    it, which is 0.23 % of the largest value, and that is under four times the values' mean here: 1 % for each of the two quantised operands of a product, and some BF16 roundings."""
    block.quantize()
    x, residual = _rows(6, tokens).cuda(), _rows(7, tokens).cuda()
    got, stream = block.decode(x, residual)
    from deepep_amd import dense, w4, w8

    layer = block.layer
    normed = dense.rms_norm(x, block.norm, residual)
    assert torch.equal(normed.stream, stream)
    topk_idx, _ = layer.router.route(normed.y.float() @ layer.gate.T, layer.bias)
    gate_up, down = (w4.dequantize(w).double().cpu() for w in layer.quantized[:2])
    parameters = [block.norm.double().cpu(), *(w8.dequantize(w).double().cpu() for w in block.shared_8), layer.gate.double().cpu(), gate_up, down]
    _near(got, _exact(block, stream.double().cpu(), topk_idx.cpu().long(), parameters), 2.5e-2, "decode")


def test_a_captured_decode_replays(block):
    block.quantize()
    x, residual = _rows(8, 4).cuda(), _rows(9, 4).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block.decode(x, residual)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, stream = block.decode(x, residual)
    for seed in (10, 11, 12, 13):
        x.copy_(_rows(seed, 4))
        residual.copy_(_rows(seed + 10, 4))
        want, want_stream = block.decode(x, residual)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(stream, want_stream)


def test_dispatch_takes_the_norms_codes():
    """Codes and scales as the norm leaves them arrive in the rows of their tokens, byte for byte."""
    from deepep_amd import ElasticBuffer, dense

    tokens, hidden, experts, topk = 70, 512, 8, 3
    gen = torch.Generator().manual_seed(14)
    x = torch.randn(tokens, hidden, generator=gen).bfloat16().cuda()
    idx = torch.stack([torch.randperm(experts, generator=gen)[:topk] for _ in range(tokens)]).cuda()
    weights = torch.rand(tokens, topk, generator=gen).cuda()
    normed = dense.rms_norm(x, torch.ones(hidden, device="cuda"), quantize="fp8", output=False)
    assert normed.y is None
    buf = ElasticBuffer(None, num_max_tokens_per_rank=tokens, hidden=hidden, num_topk=topk, use_fp8_dispatch=True, explicitly_destroy=True)
    try:
        (rows, scales), _, _, handle, _ = buf.dispatch((normed.codes, normed.scales), topk_idx=idx, topk_weights=weights, num_experts=experts, do_expand=True)
        order = torch.cat([(idx.cpu() == e).nonzero()[:, 0] for e in range(experts)])
        assert [int((idx == e).sum()) for e in range(experts)] == list(handle.num_recv_tokens_per_expert_list)
        assert torch.equal(rows.view(torch.uint8).cpu(), normed.codes.view(torch.uint8).cpu()[order]) and torch.equal(scales.cpu(), normed.scales.cpu()[order])
    finally:
        buf.destroy()


def test_mega_moe_takes_the_norms_codes():
    from deepep_amd import dense, megamoe
    from oracle import megamoe as mm
    from tests.test_gpu_megamoe import _make_problem, _oracle

    tokens, hidden, inter, experts, topk = 33, 1024, 512, 4, 2
    _, _, l1, l2, idx, weights = _make_problem(tokens, hidden, inter, experts, 0, experts, topk, seed=15)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(16)).bfloat16().cuda()
    normed = dense.rms_norm(x, torch.ones(hidden, device="cuda"), quantize="mxfp8", output=False)
    buf = megamoe.SymmBuffer(None, experts, tokens, topk, hidden, inter)
    try:
        p1, p2 = megamoe.transform_weights_for_mega_moe(*((torch.from_numpy(w).cuda(), torch.from_numpy(sc).cuda()) for w, sc in (l1, l2)))
        buf.x.view(torch.uint8).copy_(normed.codes.view(torch.uint8))
        buf.x_sf.view(torch.uint8).copy_(normed.scales)
        buf.topk_idx.copy_(torch.from_numpy(idx))
        buf.topk_weights.copy_(torch.from_numpy(weights))
        buf.validate_inputs(tokens)
        y = torch.empty((tokens, hidden), dtype=torch.bfloat16, device="cuda")
        megamoe.fp8_fp4_mega_moe(y, p1, p2, buf)
        want = _oracle(normed.codes.view(torch.uint8).cpu().numpy(), normed.scales.cpu().numpy(), l1, l2, idx, weights, 0)
        assert mm.relative_frobenius(y.float().cpu().numpy(), want) <= 2e-2
    finally:
        buf.destroy()


def test_inference_mode_and_leaves(block):
    """The same results in inference mode, of inference tensors, and of leaves that want gradients (none are recorded)."""
    from deepep_amd import dense, w8

    block.quantize()
    x, residual = _rows(17, 6).cuda(), _rows(18, 6).cuda()
    want = block.decode(x, residual)
    y, kept = dense.gated_ffn(x, block.shared_gate_up, block.shared_down, keep=True)
    grads = dense.gated_ffn_backward(residual, x, block.shared_gate_up, block.shared_down, kept)
    with torch.inference_mode():
        got = block.decode(x.clone(), residual.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(w8.matmul(x.clone(), block.shared_8[0]), w8.matmul(x, block.shared_8[0]))
        again = dense.gated_ffn_backward(residual.clone(), x.clone(), block.shared_gate_up, block.shared_down, kept.clone())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    leaves = [t.clone().requires_grad_(True) for t in (x, block.shared_gate_up, block.shared_down)]
    out = dense.gated_ffn(*leaves)
    assert torch.equal(out, y) and not out.requires_grad
