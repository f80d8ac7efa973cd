"""The gated feed-forward block on the GPU, both directions, against the 64-bit oracle within the bounds that it derives (32-bit sums, one
rounding of the rows between the products, one of the result)."""

import numpy as np
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _make(tokens, hidden, inter, dtype, seed=0):
    gen = torch.Generator().manual_seed(tokens * 7919 + hidden * 31 + inter + seed)
    make = lambda *shape, scale: (torch.randn(shape, generator=gen) * scale).to(DTYPES[dtype]).cuda()  # noqa: E731
    return (make(tokens, hidden, scale=1.0), make(2 * inter, hidden, scale=hidden**-0.5), make(hidden, inter, scale=inter**-0.5), make(tokens, hidden, scale=1.0))


def _wide(*tensors):
    return [t.double().cpu().numpy() for t in tensors]


def _check(got, want, bound):
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:5].tolist())


SIZES = [  # tokens, hidden, inter
    (1, 8, 8), (1, 256, 128), (1, 1024, 704), (2, 264, 136), (3, 72, 24), (4, 2880, 1408), (5, 512, 256), (7, 1032, 520), (8, 640, 1024), (15, 128, 264), (16, 768, 384), (17, 768, 384),
    (31, 2048, 72), (32, 80, 2048), (33, 2880, 1408), (48, 512, 512), (63, 320, 200), (64, 1024, 512), (65, 1024, 512), (100, 136, 1000), (127, 264, 128), (128, 512, 256), (129, 520, 264),
    (192, 1024, 264), (255, 264, 520), (256, 512, 512), (257, 520, 520), (300, 2048, 256), (511, 768, 768), (513, 264, 1288), (700, 1032, 256), (1000, 512, 128),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
def test_forward(tokens, hidden, inter, dtype):
    from deepep_amd import dense

    x, gate_up, down, _ = _make(tokens, hidden, inter, dtype)
    y = dense.gated_ffn(x, gate_up, down)
    assert y.dtype == x.dtype and y.shape == x.shape
    want = od.ffn(*_wide(x, gate_up, down), dtype)
    _check(y, want["y"], want["y_off"])
    # two roundings of a step's half each, spread evenly: the whole is off by no more
    off = np.linalg.norm(y.double().cpu().numpy() - want["y"]) / np.linalg.norm(want["y"])
    assert off <= np.sqrt(2 / 3) * od.HALF[dtype] + 1e-5
    kept_y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    assert torch.equal(kept_y, y) and kept.dtype == torch.float32 and kept.shape == (tokens, 2 * inter)
    _check(kept, want["z"], want["z_off"])
    assert torch.equal(y, dense.gated_ffn(x, gate_up, down))


@pytest.mark.parametrize("tokens,hidden,inter,dtype", [(*size, "bf16" if i % 3 else "fp16") for i, size in enumerate(SIZES)])
def test_backward(tokens, hidden, inter, dtype):
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(tokens, hidden, inter, dtype)
    _, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    got = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    want = od.ffn_backward(*_wide(grad_y, x, gate_up, down), dtype)
    for grad, like, (value, bound) in zip(got, (x, gate_up, down), want):
        assert grad.dtype == like.dtype and grad.shape == like.shape
        _check(grad, value, bound)
        off = np.linalg.norm(grad.double().cpu().numpy() - value) / np.linalg.norm(value)
        assert off <= np.sqrt(2 / 3) * od.HALF[dtype] + 1e-5
    for a, b in zip(got, dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,hidden,inter", [(4096, 1024, 1032), (2100, 2056, 1536)])
def test_many_tokens(tokens, hidden, inter):
    """Sizes at which the products take their largest tiles, and the three of the backward pass a launch together."""
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(tokens, hidden, inter, "bf16")
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    want = od.ffn(*_wide(x, gate_up, down), "bf16")
    _check(y, want["y"], want["y_off"])
    got = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    for grad, (value, bound) in zip(got, od.ffn_backward(*_wide(grad_y, x, gate_up, down), "bf16")):
        _check(grad, value, bound)
    for a, b in zip(got, dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)):
        assert torch.equal(a, b)


def test_gradients_match_differences():
    """The change of a loss along a direction, from the block itself in half precision, against its gradients: to 2 %, what two outputs rounded to 2^-11 leave of a
    difference of a tenth of them."""
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(24, 128, 64, "fp16")
    _, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    grads = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    for i, (t, grad) in enumerate(zip((x, gate_up, down), grads)):
        step = (grad.double() / grad.double().norm() * t.double().norm() * 0.02).half()  # a direction in which the loss changes
        moved = [[(u.double() + sign * step.double() if j == i else u.double()).half() for j, u in enumerate((x, gate_up, down))] for sign in (1, -1)]
        loss = [(dense.gated_ffn(*m).double() * grad_y.double()).sum() for m in moved]
        along = (grad.double() * (moved[0][i].double() - moved[1][i].double())).sum()
        assert abs((loss[0] - loss[1]) / along - 1) < 0.02


def test_no_tokens():
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(0, 64, 32, "bf16")
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    assert y.shape == (0, 64) and kept.shape == (0, 64)
    grad_x, grad_gate_up, grad_down = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    assert grad_x.shape == (0, 64) and not grad_gate_up.any() and not grad_down.any()


def test_values_that_are_not_finite_stay_in_their_token():
    from deepep_amd import dense

    x, gate_up, down, _ = _make(40, 264, 136, "bf16")
    want = dense.gated_ffn(x, gate_up, down)
    x[7, 3], x[20, 5] = float("nan"), float("inf")
    got = dense.gated_ffn(x, gate_up, down)
    rest = torch.tensor([t for t in range(40) if t not in (7, 20)], device="cuda")
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[7]).all() and not torch.isfinite(got[20]).any()


def test_large_gates_saturate():
    """A gate far below zero passes nothing on, one far above is passed through; no infinities on the way."""
    from deepep_amd import dense

    x = torch.ones(2, 8, dtype=torch.bfloat16, device="cuda")
    gate_up = torch.zeros(16, 8, dtype=torch.bfloat16, device="cuda")
    gate_up[:4, 0], gate_up[4:8, 0], gate_up[8:, 0] = 2000.0, -2000.0, 1.0
    down = torch.eye(8, dtype=torch.bfloat16, device="cuda")
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    assert (y[:, :4] == 2000).all() and (y[:, 4:] == 0).all()
    grads = dense.gated_ffn_backward(x, x, gate_up, down, kept)
    assert all(torch.isfinite(g).all() for g in grads)
    assert (grads[1][4:8] == 0).all() and (grads[1][12:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens", [1, 200])
def test_gates_of_all_sizes(tokens, dtype):
    """The activation and its gradients by themselves: products of one term each, which are exact, so that what is off is the 32-bit arithmetic between them (more for large gates) and one
    rounding to 16 bits."""
    from deepep_amd import dense

    size = 512
    rng = np.random.default_rng(tokens)
    gates = np.concatenate([-np.linspace(5, 80, 300), np.linspace(-5, 80, size - 300)])
    rounded = lambda v: torch.from_numpy(v).to(DTYPES[dtype]).cuda()  # noqa: E731
    x = torch.zeros(tokens, size, dtype=DTYPES[dtype], device="cuda")
    x[0, 0] = 1
    gate_up = torch.zeros(2 * size, size, dtype=DTYPES[dtype], device="cuda")
    gate_up[:size, 0], gate_up[size:, 0] = rounded(gates), rounded(rng.normal(size=size) * np.exp(np.clip(-gates, 0, 60) if dtype == "bf16" else 0 * gates))
    down = torch.eye(size, dtype=DTYPES[dtype], device="cuda")
    grad_y = torch.zeros_like(x)
    grad_y[0] = rounded(rng.normal(size=size))
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    assert torch.equal(kept[0], gate_up[:, 0].float()) and not kept[1:].any() and not y[1:].any()
    _, grad_gate_up, _ = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    g, u, dh = _wide(gate_up[:size, 0], gate_up[size:, 0], grad_y[0])
    share = 1 / (1 + np.exp(-g))
    dg, du = dh * u * share * (1 + g * (1 - share)), dh * g * share
    for got, want, off in ((y[0], g * share * u, od.h_off(g, u)), (grad_gate_up[:size, 0], dg, od.dz_off(dh, g, u)[0]), (grad_gate_up[size:, 0], du, od.dz_off(dh, g, u)[1])):
        assert (off <= 0.1 * od.HALF[dtype] * np.abs(want) + od.HALF[dtype] ** 2).all()  # (and says something)
        _check(got, want, off + od.HALF[dtype] * (np.abs(want) + off) + od.TINY[dtype])


@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_nothing_is_written_past_the_rows(tokens):
    """Results in the middle of larger buffers, through the C-ABI: what lies around them stays as it was."""
    import ctypes

    from deepep_amd import _lib, dense, ops

    hidden, inter = 264, 136
    x, gate_up, down, grad_y = _make(tokens, hidden, inter, "bf16")
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    grads = dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)
    lib, stream = _lib.load(), ops._stream(x.device)
    call = ops._Ffn(gate_up.data_ptr(), down.data_ptr(), 1, hidden, inter)

    def guarded(like):
        whole = torch.full((like.numel() + 4096,), 7, dtype=like.dtype, device="cuda")
        return whole, whole[2048 : 2048 + like.numel()].view(like.shape)

    scratch = guarded(torch.empty(max(lib.dpep_gated_ffn_scratch_bytes(tokens, hidden, inter), lib.dpep_gated_ffn_backward_scratch_bytes(tokens, hidden, inter)), dtype=torch.uint8))
    outs = [guarded(t) for t in (y, kept, *grads)]
    at = [o[1].data_ptr() for o in outs]
    assert lib.dpep_gated_ffn(ctypes.byref(call), x.data_ptr(), tokens, at[0], at[1], scratch[1].data_ptr(), stream) == 0
    assert lib.dpep_gated_ffn_backward(ctypes.byref(call), grad_y.data_ptr(), x.data_ptr(), at[1], tokens, at[2], at[3], at[4], scratch[1].data_ptr(), stream) == 0
    torch.cuda.synchronize()
    for (whole, part), want in zip(outs, (y, kept, *grads)):
        assert torch.equal(part, want)
        assert (whole[:2048] == 7).all() and (whole[2048 + part.numel():] == 7).all()
    assert (scratch[0][:2048] == 7).all() and (scratch[0][2048 + scratch[1].numel():] == 7).all()


@pytest.mark.parametrize("tokens", [1, 40, 600])
def test_a_captured_step_replays(tokens):
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(tokens, 520, 264, "bf16")

    def step():
        y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
        return [y, kept, *dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)]

    step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        more = step()
    gen = torch.Generator().manual_seed(1)
    for turn in range(3):
        x.copy_(torch.randn(x.shape, generator=gen))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, want, more):
            assert torch.equal(a, b) and torch.equal(c, b)


def test_two_streams_at_once():
    from deepep_amd import dense

    sets = [_make(300, 520, 264, "bf16", seed) for seed in (1, 2)]
    want = [dense.gated_ffn(*s[:3]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense.gated_ffn(*sets[i][:3]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_two_streams_at_once_backward():
    """The three products in one launch, on two streams with a scratch of each."""
    from deepep_amd import dense, ops

    assert all(c["together"] for c in ops.product_choices("ffn_backward", 700, 1032, 256)[1:]) and ops.product_choices("ffn_backward", 700, 1032, 256)[0]["parts"] > 1
    sets = []
    for seed in (1, 2):
        x, gate_up, down, grad_y = _make(700, 1032, 256, "bf16", seed)
        sets.append((grad_y, x, gate_up, down, dense.gated_ffn(x, gate_up, down, keep=True)[1]))
    want = [dense.gated_ffn_backward(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense.gated_ffn_backward(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for grads in got[i] for a, b in zip(grads, want[i]))


def test_unaligned_rows_and_parameters():
    from deepep_amd import dense

    x, gate_up, down, grad_y = _make(5, 264, 136, "bf16")
    y, kept = dense.gated_ffn(x, gate_up, down, keep=True)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)  # noqa: E731
    assert torch.equal(dense.gated_ffn(odd(x), odd(gate_up), odd(down)), y)
    assert torch.equal(dense.gated_ffn(x, torch.nn.Parameter(gate_up), torch.nn.Parameter(down)), y)
    for a, b in zip(dense.gated_ffn_backward(odd(grad_y), odd(x), odd(gate_up), odd(down), odd(kept)), dense.gated_ffn_backward(grad_y, x, gate_up, down, kept)):
        assert torch.equal(a, b)
