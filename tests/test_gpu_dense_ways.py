"""The feed-forward block and the 8-bit products at sizes that take each way of making a product: streams of one matrix, tiles of 128 and 256, one and two to a compute unit, k in
parts, the backward's products together and apart.  Large results are compared in some of their rows and columns, the edges of tiles among them, with the 64-bit
oracle's of just these: a token's output needs no other token, the gradients of an inner channel's weights no other channel."""

import numpy as np
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _some(count, how_many, seed):
    """Places at the edges of tiles and others."""
    edges = [0, 1, 15, 16, 63, 64, 127, 128, 255, 256, count - 256, count - 128, count - 65, count - 16, count - 1]
    drawn = np.random.default_rng(seed).integers(0, count, size=how_many).tolist()
    return sorted({i for i in edges + drawn if 0 <= i < count})


def _wide(*tensors):
    return [t.double().cpu().numpy() for t in tensors]


def _check(got, want, bound):
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:5].tolist())


SIZES = [  # tokens, hidden, inter
    (3, 4104, 2056), (16, 4504, 2312), (20, 4104, 2064), (40, 4104, 2064), (250, 2088, 1000), (500, 4104, 1032), (1001, 2888, 1400), (1500, 1032, 1408), (1600, 640, 160),
    (16000, 640, 160), (2047, 2056, 1016), (16000, 128, 4104), (103, 296, 4552), (590, 984, 3592), (6175, 912, 240), (36, 5848, 1928), (4090, 4072, 2040), (8100, 4040, 2008),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
def test_block(tokens, hidden, inter, dtype):
    from deepep_amd import dense

    gen = torch.Generator(device="cuda").manual_seed(tokens + hidden + inter)
    make = lambda *shape, scale=1.0: (torch.randn(shape, generator=gen, device="cuda") * scale).to(DTYPES[dtype])  # noqa: E731
    x, gate_up, down, grad_y = make(tokens, hidden), make(2 * inter, hidden, scale=hidden**-0.5), make(hidden, inter, scale=inter**-0.5), make(tokens, hidden, scale=tokens**-0.5)
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    grads = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    rows, inner = _some(tokens, 20, tokens), _some(inter, 12, inter)
    parameters = _wide(gate_up, down)
    of_rows = _wide(x[rows], grad_y[rows])
    want = od.ffn(of_rows[0], *parameters, dtype)
    _check(y[rows], want["y"], want["y_off"])
    _check(kept[rows], want["z"], want["z_off"])
    _check(grads[0][rows], *od.ffn_backward(of_rows[1], of_rows[0], *parameters, dtype)[0])
    both = inner + [inter + i for i in inner]
    _, of_gate_up, of_down = od.ffn_backward(*_wide(grad_y, x, gate_up[both], down[:, inner]), dtype)
    _check(grads[1][both], *of_gate_up)
    _check(grads[2][:, inner], *of_down)
    assert torch.equal(y, dense.gated_ffn(x, gate_up, down))
    for a, b in zip(grads, dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", [(5, 5001, 1008), (14, 4100, 4112), (30, 5001, 1040), (400, 1001, 7184), (1500, 2567, 1040), (3000, 1030, 400), (4100, 4099, 2064), (8200, 513, 4112), (8190, 4090, 4112)])
def test_codes(rows, n, k, dtype):
    from deepep_amd import w8

    gen = torch.Generator(device="cuda").manual_seed(rows + n + k)
    codes = lambda *shape: torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)  # noqa: E731
    scales = lambda count: (0.5 + torch.rand(count, generator=gen, device="cuda")) * 0.01  # noqa: E731
    x, w = (codes(rows, k), scales(rows)), (codes(n, k), scales(n))
    y = w8.matmul(x, w8.W8Weights(*w), dtype=DTYPES[dtype])
    some = _some(rows, 20, rows)
    a, b = _wide(x[0][some], w[0])
    want = (a @ b.T) * x[1][some].double().cpu().numpy()[:, None] * w[1].double().cpu().numpy()  # (whole numbers under 2^53)
    # the sum as a 32-bit number and two products of it: three roundings, then the result's
    bound = 4 * od.EPS32 * np.abs(want)
    _check(y[some], want, bound + od.HALF[dtype] * (np.abs(want) + bound) + od.TINY[dtype])
    assert torch.equal(y, w8.matmul(x, w8.W8Weights(*w), dtype=DTYPES[dtype]))
