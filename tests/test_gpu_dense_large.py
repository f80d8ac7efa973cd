"""The norm, the feed-forward block and the 8-bit products with tensors of more than 2^31 values: rows at both ends against the oracle, or against the same rows among fewer.
Everything between is zeros, which add nothing to a gradient."""

import numpy as np
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu


def _wide(*tensors):
    return [t.double().cpu().numpy() for t in tensors]


def _check(got, want, bound):
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:5].tolist())


def _ends(rows, columns, gen, few=150):
    """BF16 zeros with random rows at both ends, and which rows those are."""
    x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    some = list(range(few)) + list(range(rows - few, rows))
    x[:few], x[-few:] = (torch.randn(few, columns, generator=gen, device="cuda").bfloat16() for _ in range(2))
    return x, some


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("quantize", ["fp8", "mxfp8", "int8"])
def test_norm(quantize):
    from deepep_amd import dense

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, some = _ends(270_000, 8192, gen)
    w = torch.randn(8192, generator=gen, device="cuda")
    got, want = dense.rms_norm(x, w, x, quantize=quantize), dense.rms_norm(x[some], w, x[some], quantize=quantize)
    for a, b in zip(got, want):
        assert torch.equal(a[some].view(torch.uint8), b.view(torch.uint8))
    if quantize == "int8":
        grad_x, grad_weight = dense.rms_norm_backward(x, got.stream, w, got.rstd, x)
        few_x, few_weight = dense.rms_norm_backward(x[some], want.stream, w, want.rstd, x[some])
        assert torch.equal(grad_x[some], few_x)
        # the same 300 numbers of a column in another order
        terms = (x[some].double() * want.stream.double() * want.rstd.double()[:, None]).abs().sum(0)
        assert ((grad_weight - few_weight).double().abs() <= 300 * od.EPS32 * terms).all()


@pytest.mark.parametrize("tokens,hidden,inter", [(270_000, 8192, 64), (20_000, 64, 65536)])
def test_block(tokens, hidden, inter):
    from deepep_amd import dense

    gen = torch.Generator(device="cuda").manual_seed(2)
    x, some = _ends(tokens, hidden, gen)
    grad_y, _ = _ends(tokens, hidden, gen)
    gate_up, down = ((torch.randn(shape, generator=gen, device="cuda") * shape[1] ** -0.5).bfloat16() for shape in ((2 * inter, hidden), (hidden, inter)))
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    grads = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    few, parameters = _wide(x[some], grad_y[some]), _wide(gate_up, down)
    want = od.ffn(few[0], *parameters, "bf16")
    _check(y[some], want["y"], want["y_off"])
    _check(kept[some], want["z"], want["z_off"])
    of_x, of_gate_up, of_down = od.ffn_backward(few[1], few[0], *parameters, "bf16")
    _check(grads[0][some], *of_x)
    _check(grads[1], *of_gate_up)
    _check(grads[2], *of_down)
    assert not y[150:-150].any() and not grads[0][150:-150].any()


@pytest.mark.parametrize("rows,n,k", [(270_000, 8201, 16), (40_000, 24, 65536), (24, 40_000, 65536)])
def test_products(rows, n, k):
    from deepep_amd import w8

    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.zeros(count, k, dtype=torch.int8, device="cuda") for count in (rows, n))
    for t in (x, w):
        part = min(200, t.shape[0])
        for at in (slice(0, part), slice(t.shape[0] - part, t.shape[0])):
            t[at] = torch.randint(-127, 128, (part, k), generator=gen, device="cuda", dtype=torch.int8)
    x_scales, w_scales = (0.5 + torch.rand(count, generator=gen, device="cuda") for count in (rows, n))
    y = w8.matmul((x, x_scales), w8.W8Weights(w, w_scales))
    ends = [sorted(set(range(min(count, 200))) | set(range(max(count - 200, 0), count))) for count in (rows, n)]
    a, b = _wide(x[ends[0]], w[ends[1]])
    want = (a @ b.T) * x_scales[ends[0]].double().cpu().numpy()[:, None] * w_scales[ends[1]].double().cpu().numpy()
    bound = 4 * od.EPS32 * np.abs(want)
    _check(y[ends[0]][:, ends[1]], want, bound + od.HALF["bf16"] * (np.abs(want) + bound) + od.TINY["bf16"])
    assert not y[200:-200].any() if rows > 400 else True
