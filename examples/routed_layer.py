"""A mixture-of-experts layer from the gate's logits on: a few training steps, then decoding with its weights in 4 bits.  And a layer as a model has
it: the residual's addition and the norm in front, a shared expert beside.

    python -m examples.routed_layer

Training: gate logits -> ``Router.route_with_balance`` -> ``ElasticBuffer.dispatch`` -> experts -> ``combine``, and back; ``combine`` returns
the gradient of the route weights, from which ``Router.backward`` makes that of the logits, the balance loss's share in the same pass.  The counts
of the balance loss also move the bias that spreads the choice.  Decoding: ``Router.route`` -> ``w4.expert_ffn``, beside them a shared expert
through ``w4.matvec``, no dispatch.  ``Block`` puts ``dense.rms_norm`` in front of the layer and ``dense.gated_ffn`` beside it, with their gradients;
it serves from ``dense.rms_norm(quantize="int8")`` through ``w8.matmul``, whose weights are held in 8 bits.  Data and weights are random; experts are plain torch, which is not what this is about.
"""

import torch
import torch.nn.functional as F

from deepep_amd import ElasticBuffer, Router, dense, w4, w8


def expert_rows(rows, counts, gate_up, down):
    """SwiGLU experts over rows that are sorted by expert."""
    out = []
    for e, part in enumerate(rows.split(counts)):
        gate, up = (part @ gate_up[e].T).chunk(2, dim=1)
        out.append((F.silu(gate) * up) @ down[e].T)
    return torch.cat(out)


class RoutedLayer:
    def __init__(self, hidden, inter, experts, topk, *, max_tokens, groups=1, topk_groups=1, scale=1.0, device="cuda", seed=0):
        gen = torch.Generator().manual_seed(seed)

        def weights(*shape):
            return (torch.randn(*shape, generator=gen) / shape[-1] ** 0.5).to(device)

        self.experts = experts
        self.gate = weights(experts, hidden)
        self.gate_up, self.down = weights(experts, 2 * inter, hidden), weights(experts, hidden, inter)
        self.shared_gate_up, self.shared_down = weights(2 * inter, hidden), weights(hidden, inter)
        self.bias = torch.zeros(experts, device=device)
        self.router = Router(experts, topk, score="sigmoid", scale=scale, num_groups=groups, num_topk_groups=topk_groups)
        self.buffer = ElasticBuffer(None, num_max_tokens_per_rank=max_tokens, hidden=hidden, num_topk=topk, explicitly_destroy=True)

    # ---- training ----------------------------------------------------------------------------------------------------------------
    def forward(self, x, token_mask=None, sequence_offsets=None):
        """x BF16 [T,H]: the routed experts' output BF16 [T,H], the balance loss, and what ``backward`` needs."""
        logits = x.float() @ self.gate.T
        topk_idx, topk_weights, balance = self.router.route_with_balance(logits, self.bias, token_mask, sequence_offsets=sequence_offsets)
        rows, _, row_weights, handle, _ = self.buffer.dispatch(x, topk_idx=topk_idx, topk_weights=topk_weights, num_experts=self.experts, do_expand=True)
        with torch.enable_grad():
            leaves = [t.detach().float().requires_grad_(True) for t in (rows, row_weights, self.gate_up, self.down)]
            row_out = expert_rows(leaves[0], handle.num_recv_tokens_per_expert_list, leaves[2], leaves[3]) * leaves[1][:, None]
        out, _, _ = self.buffer.combine(row_out.detach().bfloat16(), handle)
        return out, balance, (x, logits, topk_idx, topk_weights, balance, handle, leaves, row_out)

    def backward(self, grad_out, saved, balance_weight=0.0):
        """Gradients of x, the gate and the experts' weights for ``grad_out`` BF16 [T,H] and ``balance_weight`` times the mean balance loss."""
        x, logits, topk_idx, topk_weights, balance, handle, leaves, row_out = saved
        grad_rows_out = self.buffer.dispatch(grad_out, handle=handle)[0]
        grad_rows, grad_row_weights, grad_gate_up, grad_down = torch.autograd.grad(row_out, leaves, grad_rows_out.float())
        grad_x, grad_weights, _ = self.buffer.combine(grad_rows.bfloat16(), handle, topk_weights=grad_row_weights.contiguous())
        grad_losses = torch.full_like(balance.losses, balance_weight / balance.losses.numel())
        grad_logits = self.router.backward(logits, topk_idx, topk_weights=topk_weights, grad_weights=grad_weights, balance=balance, grad_losses=grad_losses)
        grad_x = grad_x.float() + grad_logits @ self.gate
        return grad_x, grad_logits.T @ x.float(), grad_gate_up, grad_down

    def move_bias(self, balance, rate):
        """Towards experts with fewer routes than their share, away from those with more."""
        counts = balance.counts.sum(dim=0).float()
        self.bias += rate * torch.sign(counts.mean() - counts)

    # ---- decoding ----------------------------------------------------------------------------------------------------------------
    def quantize(self, group=64):
        weights = (self.gate_up, self.down, self.shared_gate_up, self.shared_down)
        self.quantized = [w4.quantize(w, group, symmetric=False) for w in weights]

    def decode(self, x):
        """x BF16 [T,H] of a few tokens: routed and shared experts' output BF16 [T,H]."""
        gate_up, down, shared_gate_up, shared_down = self.quantized
        topk_idx, topk_weights = self.router.route(x.float() @ self.gate.T, self.bias)
        gate, up = w4.matvec(x, shared_gate_up).chunk(2, dim=1)
        return w4.expert_ffn(x, topk_idx, topk_weights, gate_up, down) + w4.matvec((F.silu(gate) * up).contiguous(), shared_down)

    def destroy(self):
        self.buffer.destroy()


class Block:
    """stream = x + residual; normed = norm(stream); routed experts(normed) + shared expert(normed).  The stream goes on to the next block."""

    def __init__(self, layer):
        self.layer = layer
        self.norm = torch.ones(layer.gate.shape[1], device=layer.gate.device)
        self.shared_gate_up, self.shared_down = layer.shared_gate_up.bfloat16(), layer.shared_down.bfloat16()

    def forward(self, x, residual, token_mask=None, sequence_offsets=None):
        """x, residual BF16 [T,H]: output and stream BF16 [T,H], the balance loss, and what ``backward`` needs."""
        normed = dense.rms_norm(x, self.norm, residual)
        routed, balance, saved = self.layer.forward(normed.y, token_mask, sequence_offsets)
        shared, kept = dense.gated_ffn(normed.y, self.shared_gate_up, self.shared_down, keep=True)
        return routed + shared, normed.stream, balance, (normed, saved, kept)

    def backward(self, grad_out, grad_stream, saved, balance_weight=0.0):
        """Gradients of x (and of the residual, which is the same), the norm, the shared expert's matrices, the gate and the experts' matrices."""
        normed, of_layer, kept = saved
        grad_routed, *grads = self.layer.backward(grad_out, of_layer, balance_weight)
        grad_shared, *shared_grads = dense.gated_ffn_backward(grad_out, normed.y, self.shared_gate_up, self.shared_down, kept)
        grad_x, grad_norm = dense.rms_norm_backward((grad_routed + grad_shared).bfloat16(), normed.stream, self.norm, normed.rstd, grad_stream)
        return grad_x, grad_norm, *shared_grads, *grads

    def quantize(self):
        self.layer.quantize()
        self.shared_8 = w8.quantize(self.shared_gate_up), w8.quantize(self.shared_down)

    def decode(self, x, residual):
        """x, residual BF16 [T,H] of a few tokens: output and stream BF16 [T,H], with routed experts in 4 bits, the shared one in 8."""
        normed = dense.rms_norm(x, self.norm, residual, quantize="int8")
        gate_up, down = self.layer.quantized[:2]
        topk_idx, topk_weights = self.layer.router.route(normed.y.float() @ self.layer.gate.T, self.layer.bias)
        gate, up = w8.matmul((normed.codes, normed.scales), self.shared_8[0]).chunk(2, dim=1)
        return w4.expert_ffn(normed.y, topk_idx, topk_weights, gate_up, down) + w8.matmul((F.silu(gate) * up).contiguous(), self.shared_8[1]), normed.stream


def main():
    tokens, hidden, steps = 1024, 512, 20
    layer = RoutedLayer(hidden, 256, 32, 4, max_tokens=tokens, groups=4, topk_groups=2, scale=2.5)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(tokens, hidden, generator=gen).cuda().bfloat16()
    target = torch.randn(tokens, hidden, generator=gen).cuda() @ torch.randn(hidden, hidden, generator=gen).cuda() / hidden
    token_mask = (torch.rand(tokens, generator=gen) > 0.1).cuda()
    offsets = torch.tensor([0, 100, 700, tokens], dtype=torch.int32).cuda()
    real = token_mask[:, None]
    for step in range(steps):
        out, balance, saved = layer.forward(x, token_mask, offsets)
        error = (out.float() - target) * real
        loss = error.square().sum() / tokens
        _, *grads = layer.backward((2 / tokens * error).bfloat16(), saved, balance_weight=0.01)
        for weight, grad in zip((layer.gate, layer.gate_up, layer.down), grads):
            weight -= 0.2 * grad
        layer.move_bias(balance, 1e-3)
        if step % 5 == 0 or step == steps - 1:
            print(f"step {step}: loss {loss.item():.3f}, balance {balance.losses.mean().item():.4f}, "
                  f"routes of an expert {balance.counts.sum(0).min().item()} to {balance.counts.sum(0).max().item()}", flush=True)
    block, residual = Block(layer), torch.randn(tokens, hidden, generator=gen).cuda().bfloat16()
    for step in range(steps):
        out, _, balance, saved = block.forward(x, residual, token_mask, offsets)
        error = (out.float() - target) * real
        _, grad_norm, grad_gate_up, grad_down, *_ = block.backward((2 / tokens * error).bfloat16(), None, saved)
        for weight, grad in ((block.norm, grad_norm), (block.shared_gate_up, grad_gate_up), (block.shared_down, grad_down)):
            weight -= 0.2 * grad
        if step % 10 == 0 or step == steps - 1:
            print(f"block, step {step}: loss {(error.square().sum() / tokens).item():.3f}", flush=True)
    block.quantize()
    few = x[:4]
    exact = block.forward(few, residual[:4])[0].float()
    got = block.decode(few, residual[:4])[0].float()
    print(f"block: 4 tokens in 4 and 8 bits differ from BF16 weights by {((got - exact).norm() / exact.norm()).item():.3f} of their norm")
    routed, _, _ = layer.forward(few)
    gate, up = (few.float() @ layer.shared_gate_up.T).chunk(2, dim=1)
    exact = routed.float() + (F.silu(gate) * up) @ layer.shared_down.T
    got = layer.decode(few).float()
    print(f"decode: 4 tokens in 4 bits differ from FP32 weights by {((got - exact).norm() / exact.norm()).item():.3f} of their norm")
    layer.destroy()


if __name__ == "__main__":
    main()
