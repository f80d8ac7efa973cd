"""The example's layer end to end: its training step against a dense model in 64 bits differentiated by autograd (tolerance of BF16
interfaces, as for the training recipe), and decoding with 4-bit weights against the same weights dequantised."""

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

TOKENS, HIDDEN, INTER, EXPERTS, TOPK = 120, 256, 128, 16, 3


@pytest.fixture
def layer():
    from examples.routed_layer import RoutedLayer

    made = RoutedLayer(HIDDEN, INTER, EXPERTS, TOPK, max_tokens=TOKENS, groups=4, topk_groups=2, scale=2.5, seed=5)
    yield made
    made.destroy()


def _near(got, want, what):
    got, want = got.double().cpu(), want.double()
    err = ((got - want).norm() / want.norm()).item()
    assert err <= 1e-2, (what, err)


def test_training_step(layer):
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(TOKENS, HIDDEN, generator=gen).bfloat16()
    grad_out = torch.randn(TOKENS, HIDDEN, generator=gen).bfloat16()
    token_mask = torch.rand(TOKENS, generator=gen) > 0.2
    cuts = [0, 1, 50, TOKENS]
    balance_weight = 30.0
    layer.bias += torch.randn(EXPERTS, generator=gen).cuda() / 16

    out, balance, saved = layer.forward(x.cuda(), token_mask.cuda(), torch.tensor(cuts, dtype=torch.int32).cuda())
    grads = layer.backward(grad_out.cuda(), saved, balance_weight=balance_weight)
    topk_idx = saved[2].cpu()
    assert torch.equal((topk_idx >= 0).all(dim=1), token_mask) and torch.equal((topk_idx >= 0).any(dim=1), token_mask)

    xr, gate, gate_up, down = (t.detach().double().cpu().requires_grad_(True) for t in (x, layer.gate, layer.gate_up, layer.down))
    scores = torch.sigmoid(xr @ gate.T)
    picked = scores.gather(1, topk_idx.clamp_min(0))
    weights = 2.5 * picked / picked.sum(dim=1, keepdim=True)
    want = torch.zeros(TOKENS, HIDDEN, dtype=torch.float64)
    for e in range(EXPERTS):
        for s in range(TOPK):
            chosen = (topk_idx[:, s] == e).nonzero()[:, 0]
            g, u = (xr[chosen] @ gate_up[e].T).chunk(2, dim=1)
            want = want.index_add(0, chosen, weights[chosen, s, None] * ((F.silu(g) * u) @ down[e].T))
    losses = []
    for begin, end in zip(cuts, cuts[1:]):
        real = token_mask[begin:end]
        counts = torch.bincount(topk_idx[begin:end][real].flatten(), minlength=EXPERTS).double()
        p = (scores / scores.sum(dim=1, keepdim=True))[begin:end][real]
        losses.append((counts * EXPERTS / counts.sum().clamp_min(1) * p.sum(dim=0)).sum() / max(int(real.sum()), 1))
    total = (want * grad_out.double()).sum() + balance_weight * sum(losses) / len(losses)
    total.backward()
    _near(out, want.detach(), "out")
    _near(balance.losses, torch.stack(losses).detach(), "losses")
    for got, leaf, name in zip(grads, (xr, gate, gate_up, down), ("x", "gate", "gate_up", "down")):
        _near(got, leaf.grad, name)


@pytest.mark.parametrize("tokens", [1, 5])
def test_decode(layer, tokens):
    from deepep_amd import w4

    gen = torch.Generator().manual_seed(7)
    x = torch.randn(tokens, HIDDEN, generator=gen).cuda().bfloat16()
    layer.quantize()
    got = layer.decode(x)
    layer.gate_up, layer.down, shared_gate_up, shared_down = (w4.dequantize(w) for w in layer.quantized)
    routed, _, _ = layer.forward(x)
    gate, up = (x.double() @ shared_gate_up.double().T).chunk(2, dim=1)
    _near(got, (routed.double() + (F.silu(gate) * up) @ shared_down.double().T).cpu(), "decode")


def test_runs(capsys):
    from examples.routed_layer import main

    main()
    lines = capsys.readouterr().out.splitlines()
    losses = [float(line.split("loss ")[1].split(",")[0]) for line in lines if line.startswith("step")]
    assert losses[-1] < losses[0]
    assert float(lines[-1].split(" by ")[1].split()[0]) < 0.2  # steps of 1/15 of a group's range, some 10 % of its norm, four matrices deep
