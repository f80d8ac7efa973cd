"""4-bit products on the GPU against the 64-bit oracle, within the bound that the oracle derives (fp32 sums in groups) plus half a last
place of the output's type."""

import numpy as np
import pytest
import torch

from oracle import w4 as ow4

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PLACE = {"bf16": 2.0**-8, "fp16": 2.0**-10}


def _weights(rng, shape, group, zeros, dtype):
    """(device triple, host triple) of random codes, all sixteen of them, and scales that differ from group to group."""
    n_k = shape
    packed = rng.integers(0, 256, size=(*n_k[:-1], n_k[-1] // 2)).astype(np.uint8)
    scales = torch.from_numpy(0.02 * (0.25 + rng.random((*n_k[:-1], n_k[-1] // group)))).to(DTYPES[dtype])
    points = rng.integers(0, 16, size=scales.shape).astype(np.uint8) if zeros else None
    device = (torch.from_numpy(packed).cuda(), scales.cuda(), None if points is None else torch.from_numpy(points).cuda())
    return device, (packed, scales.double().numpy(), points)


def _rows(rng, shape, dtype):
    x = torch.from_numpy(rng.normal(size=shape)).to(DTYPES[dtype])
    return x.cuda(), x.double().numpy()


def _check(got, want, bound, dtype):
    off = np.abs(got.double().cpu().numpy() - want)
    bound = bound + PLACE[dtype] * np.abs(want) + 6e-8
    assert (off <= bound).all(), float((off / bound).max())


MATVEC = [
    # rows, n, k, group, zeros, dtype
    (1, 1, 32, 32, False, "bf16"), (1, 16, 128, 128, False, "bf16"), (1, 4096, 7168, 128, False, "bf16"), (2, 33, 96, 32, True, "fp16"),
    (3, 17, 192, 64, False, "bf16"), (4, 100, 640, 128, True, "bf16"), (5, 40, 1408, 64, True, "fp16"), (7, 15, 288, 32, True, "bf16"),
    (8, 257, 512, 256, False, "fp16"), (9, 64, 1024, 1024, False, "bf16"), (13, 31, 448, 64, False, "fp16"), (16, 129, 2880, 32, True, "fp16"),
    (17, 80, 8192, 128, False, "bf16"), (33, 65, 2880, 64, True, "bf16"), (64, 48, 7168, 128, False, "bf16"), (65, 20, 416, 32, False, "bf16"),
    (130, 16, 256, 128, True, "fp16"), (6, 24, 16384, 128, False, "bf16"),
]


@pytest.mark.parametrize("rows,n,k,group,zeros,dtype", MATVEC)
def test_matvec(rows, n, k, group, zeros, dtype):
    from deepep_amd import w4

    rng = np.random.default_rng(rows * 1000 + k)
    device, host = _weights(rng, (n, k), group, zeros, dtype)
    x, wide = _rows(rng, (rows, k), dtype)
    y = w4.matvec(x, w4.W4Weights(*device))
    assert y.dtype == x.dtype and y.shape == (rows, n)
    _check(y, *ow4.product(wide, host), dtype)
    assert torch.equal(y, w4.matvec(x, w4.W4Weights(*device), out=torch.empty_like(y)))


EXPERTS = [
    # tokens, hidden, inter, topk, experts, group, zeros, dtype, masked, begin, index
    (1, 128, 128, 1, 1, 128, False, "bf16", 0.0, 0, torch.int64), (1, 7168, 256, 8, 16, 128, False, "bf16", 0.0, 0, torch.int64),
    (1, 512, 320, 3, 8, 64, True, "fp16", 0.0, 4, torch.int32), (2, 256, 96, 2, 4, 32, True, "bf16", 0.0, 0, torch.int64),
    (5, 320, 160, 4, 32, 32, False, "fp16", 0.2, 0, torch.int64), (16, 384, 128, 8, 24, 128, False, "bf16", 0.1, 8, torch.int64),
    (40, 256, 192, 4, 4, 64, True, "bf16", 0.0, 0, torch.int32), (64, 128, 64, 2, 2, 32, False, "bf16", 0.3, 0, torch.int64),
    (33, 192, 1408, 1, 3, 64, False, "fp16", 0.0, 1, torch.int64), (256, 128, 128, 8, 9, 64, True, "bf16", 0.05, 0, torch.int64),
    (3, 256, 128, 32, 1024, 128, False, "bf16", 0.0, 0, torch.int64), (7, 160, 4096, 2, 5, 32, True, "bf16", 0.0, 0, torch.int64),
]


@pytest.mark.parametrize("tokens,hidden,inter,topk,experts,group,zeros,dtype,masked,begin,index", EXPERTS)
def test_experts(tokens, hidden, inter, topk, experts, group, zeros, dtype, masked, begin, index):
    """begin: the first experts that are held elsewhere, as on one rank of several; masked: routes without an expert."""
    from deepep_amd import w4

    rng = np.random.default_rng(tokens * 1000 + hidden)
    local = experts - begin
    gate_up, gate_up_host = _weights(rng, (local, 2 * inter, hidden), group, zeros, dtype)
    down, down_host = _weights(rng, (local, hidden, inter), group, zeros, dtype)
    x, wide = _rows(rng, (tokens, hidden), dtype)
    x, wide = x * 0.25, wide * 0.25  # (a power of two: the same values on both sides)
    ids = np.argsort(rng.random((tokens, experts)), axis=1)[:, :topk]
    ids[rng.random(ids.shape) < masked] = -1
    if tokens > 4:
        ids[3] = -1  # a token without any route
    route_weights = rng.random((tokens, topk)).astype(np.float32)
    y = w4.expert_ffn(x, torch.from_numpy(ids).to(index).cuda(), torch.from_numpy(route_weights).cuda(), w4.W4Weights(*gate_up), w4.W4Weights(*down),
                      expert_begin=begin)
    assert y.dtype == x.dtype and y.shape == (tokens, hidden)
    want, bound = ow4.experts(wide, ids, route_weights.astype(np.float64), gate_up_host, down_host, begin)
    _check(y, want, bound, dtype)
    if tokens > 4:
        assert not y[3].any()
    again = w4.expert_ffn(x, torch.from_numpy(ids).to(index).cuda(), torch.from_numpy(route_weights).cuda(), w4.W4Weights(*gate_up), w4.W4Weights(*down),
                          expert_begin=begin, out=torch.full_like(y, float("nan")))
    assert torch.equal(y, again)


# Long rows, of which LDS holds fewer than a pass could take: in halves and all of it, one block of rows and several passes.
@pytest.mark.parametrize("rows,n,k,group,zeros,dtype", [
    (20, 48, 8192, 128, False, "bf16"), (64, 40, 7168, 128, True, "fp16"), (12, 33, 8192, 256, False, "bf16"), (6, 65, 8192, 64, True, "bf16"),
    (9, 64, 16384, 64, True, "bf16"), (70, 20, 16384, 32, False, "fp16"), (5, 2, 16384, 16384, False, "bf16"), (17, 16, 4096, 128, False, "fp16"),
])
def test_matvec_of_long_rows(rows, n, k, group, zeros, dtype):
    test_matvec(rows, n, k, group, zeros, dtype)


@pytest.mark.parametrize("tokens,hidden,inter,topk,experts,group,zeros,dtype", [
    (24, 7168, 64, 2, 2, 64, False, "bf16"), (12, 8192, 128, 1, 1, 128, True, "bf16"), (6, 8192, 64, 1, 2, 32, True, "fp16"),
    (10, 128, 8192, 1, 2, 128, False, "fp16"), (30, 128, 4096, 2, 3, 64, True, "bf16"),
])
def test_experts_of_long_rows(tokens, hidden, inter, topk, experts, group, zeros, dtype):
    test_experts(tokens, hidden, inter, topk, experts, group, zeros, dtype, 0.1, 0, torch.int64)


def test_one_expert_twice_in_a_token():
    from deepep_amd import w4

    rng = np.random.default_rng(8)
    gate_up, gate_up_host = _weights(rng, (3, 256, 128), 128, False, "bf16")
    down, down_host = _weights(rng, (3, 128, 128), 128, False, "bf16")
    x, wide = _rows(rng, (2, 128), "bf16")
    ids, route_weights = np.array([[1, 1], [2, 1]]), rng.random((2, 2)).astype(np.float32)
    y = w4.expert_ffn(x, torch.from_numpy(ids).cuda(), torch.from_numpy(route_weights).cuda(), w4.W4Weights(*gate_up), w4.W4Weights(*down))
    _check(y, *ow4.experts(wide, ids, route_weights.astype(np.float64), gate_up_host, down_host), "bf16")


def test_large_and_small_magnitudes():
    """BF16 rows beyond FP16's range, and rows with a large common offset (the sum over a group is then far from zero)."""
    from deepep_amd import w4

    rng = np.random.default_rng(9)
    device, host = _weights(rng, (64, 512), 128, False, "bf16")
    for scale, offset in ((1e30, 0.0), (1e-30, 0.0), (1.0, 50.0)):
        x = torch.from_numpy(scale * (rng.normal(size=(3, 512)) + offset)).bfloat16()
        want, bound = ow4.product(x.double().numpy(), host)
        y = w4.matvec(x.cuda(), w4.W4Weights(*device)).double().cpu().numpy()
        assert (np.abs(y - want) <= bound + 2.0**-8 * np.abs(want)).all()


def test_weights_past_two_gib_of_offsets():
    """Expert matrices whose byte offsets pass 32 bits."""
    from deepep_amd import w4

    experts, inter, hidden = 300, 1024, 7168
    gate_up = torch.empty((experts, 2 * inter, hidden // 2), dtype=torch.uint8, device="cuda")
    down = torch.empty((experts, hidden, inter // 2), dtype=torch.uint8, device="cuda")
    assert gate_up.numel() > 2**31
    rng = np.random.default_rng(10)
    last, last_host = _weights(rng, (1, 2 * inter, hidden), 128, False, "bf16")
    down_last, down_host = _weights(rng, (1, hidden, inter), 128, False, "bf16")
    gate_up[-1], down[-1] = last[0][0], down_last[0][0]
    scales, down_scales = last[1].expand(experts, -1, -1).contiguous(), down_last[1].expand(experts, -1, -1).contiguous()
    x, wide = _rows(rng, (2, hidden), "bf16")
    route_weights = np.ones((2, 1), dtype=np.float32)
    ids = np.full((2, 1), experts - 1)
    y = w4.expert_ffn(x, torch.from_numpy(ids).cuda(), torch.from_numpy(route_weights).cuda(), w4.W4Weights(gate_up, scales), w4.W4Weights(down, down_scales))
    want, bound = ow4.experts(wide, np.zeros((2, 1), dtype=int), route_weights, last_host, down_host)
    _check(y, want, bound, "bf16")


def test_empty_inputs_other_streams_and_odd_addresses():
    from deepep_amd import w4

    rng = np.random.default_rng(11)
    device, _ = _weights(rng, (40, 256), 64, True, "bf16")
    weights = w4.W4Weights(*device)
    assert w4.matvec(torch.empty((0, 256), dtype=torch.bfloat16, device="cuda"), weights).shape == (0, 40)
    gate_up, down = w4.W4Weights(*_weights(rng, (4, 128, 256), 64, False, "bf16")[0]), w4.W4Weights(*_weights(rng, (4, 256, 64), 64, False, "bf16")[0])
    empty = w4.expert_ffn(torch.empty((0, 256), dtype=torch.bfloat16, device="cuda"), torch.empty((0, 2), dtype=torch.int64, device="cuda"),
                          torch.empty((0, 2), device="cuda"), gate_up, down)
    assert empty.shape == (0, 256)
    x, _ = _rows(rng, (3, 256), "bf16")
    ids = torch.tensor([[0, 1], [3, 2], [-1, 1]]).cuda()
    route_weights = torch.rand((3, 2), device="cuda")
    want = w4.matvec(x, weights), w4.expert_ffn(x, ids, route_weights, gate_up, down)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        shifted = torch.empty(3 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 256)
        shifted.copy_(x)
        odd_scales = torch.empty(weights.scales.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(weights.scales.shape)
        odd_scales.copy_(weights.scales)
        got = w4.matvec(shifted, weights._replace(scales=odd_scales)), w4.expert_ffn(shifted, ids, route_weights, gate_up, down)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_graph_replays():
    from deepep_amd import w4

    rng = np.random.default_rng(12)
    gate_up, down = w4.W4Weights(*_weights(rng, (16, 256, 512), 128, False, "bf16")[0]), w4.W4Weights(*_weights(rng, (16, 512, 128), 128, False, "bf16")[0])
    x, ids, route_weights = torch.randn((6, 512), device="cuda").bfloat16(), torch.randint(0, 16, (6, 4), device="cuda"), torch.rand((6, 4), device="cuda")

    def step():
        return w4.expert_ffn(x, ids, route_weights, gate_up, down), w4.matvec(x, w4.W4Weights(gate_up.packed[0], gate_up.scales[0]))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for _ in range(4):
        x.copy_(torch.randn((6, 512), device="cuda"))
        ids.copy_(torch.randint(-1, 16, (6, 4), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_refusals():
    from deepep_amd import w4

    rng = np.random.default_rng(13)
    weights = w4.W4Weights(*_weights(rng, (40, 256), 64, True, "bf16")[0])
    x = torch.zeros((3, 256), dtype=torch.bfloat16, device="cuda")
    gate_up, down = w4.W4Weights(*_weights(rng, (4, 128, 256), 64, False, "bf16")[0]), w4.W4Weights(*_weights(rng, (4, 256, 64), 64, False, "bf16")[0])
    ids, route_weights = torch.zeros((3, 2), dtype=torch.int64, device="cuda"), torch.zeros((3, 2), device="cuda")
    bad = [
        lambda: w4.matvec(x.float(), weights),
        lambda: w4.matvec(x.half(), weights),
        lambda: w4.matvec(x.cpu(), weights),
        lambda: w4.matvec(x[:, :128], weights),
        lambda: w4.matvec(x[0], weights),
        lambda: w4.matvec(x, weights._replace(packed=weights.packed.view(torch.int8))),
        lambda: w4.matvec(x, weights._replace(packed=weights.packed[None])),
        lambda: w4.matvec(x, weights._replace(scales=weights.scales[:, :3].contiguous())),
        lambda: w4.matvec(x, weights._replace(scales=weights.scales[:39])),
        lambda: w4.matvec(x, weights._replace(zeros=weights.zeros[:, :2].contiguous())),
        lambda: w4.matvec(x, weights, out=torch.zeros((3, 41), dtype=torch.bfloat16, device="cuda")),
        lambda: w4.matvec(x, w4.W4Weights(torch.zeros((40 * 128 + 1,), dtype=torch.uint8, device="cuda")[1:].view(40, 128), weights.scales)),
        lambda: w4.expert_ffn(x, ids, route_weights, gate_up, gate_up),
        lambda: w4.expert_ffn(x, ids.float(), route_weights, gate_up, down),
        lambda: w4.expert_ffn(x, ids[:2], route_weights, gate_up, down),
        lambda: w4.expert_ffn(x, ids, route_weights.double(), gate_up, down),
        lambda: w4.expert_ffn(x, ids, route_weights, gate_up, down._replace(scales=down.scales.half())),
        lambda: w4.expert_ffn(x, ids, route_weights, gate_up, down, expert_begin=-1),
        lambda: w4.expert_ffn(x[:1].expand(1025, -1).contiguous(), ids[:1].expand(1025, -1).contiguous(), route_weights[:1].expand(1025, -1).contiguous(), gate_up, down),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_native_and_python_layers_agree():
    """Rows that carry a gradient go through the Python layer; the bits are the same."""
    from deepep_amd import _lib, w4

    rng = np.random.default_rng(14)
    gate_up, down = w4.W4Weights(*_weights(rng, (6, 192, 256), 64, True, "bf16")[0]), w4.W4Weights(*_weights(rng, (6, 256, 96), 32, False, "bf16")[0])
    x = torch.randn((4, 256), device="cuda").bfloat16()
    ids, route_weights = torch.randint(0, 6, (4, 3), device="cuda"), torch.rand((4, 3), device="cuda")
    matrix = w4.W4Weights(gate_up.packed[1], gate_up.scales[1], gate_up.zeros[1])
    assert _lib.host().w4_matvec(x, *matrix, None) is not None
    leaf = x.clone().requires_grad_()
    assert _lib.host().w4_matvec(leaf, *matrix, None) is None
    assert torch.equal(w4.matvec(leaf, matrix), w4.matvec(x, matrix))
    assert torch.equal(w4.expert_ffn(leaf, ids, route_weights, gate_up, down), w4.expert_ffn(x, ids, route_weights, gate_up, down))


@pytest.mark.parametrize("rows,n,k", [(16, 17, 8192), (16, 129, 4096), (33, 65, 8192), (1, 4097, 7168), (64, 31, 2048), (4, 1407, 2816), (3, 250, 16384)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_columns_of_a_matrix_that_ends_inside_a_tile(rows, n, k, dtype):
    """The bits are those of the same columns of a matrix of whole tiles.  Eight parts of k cancel (the same weights, whole numbers that add up to
    zero), so a result is what its sums in 32 bits left over, and any other order of them shows."""
    from deepep_amd import w4

    rng = np.random.default_rng(n + k)
    whole = -(-n // 16) * 16
    parts = [rng.integers(-15, 16, size=(rows, k // 8)) for _ in range(7)]
    x = torch.from_numpy(np.concatenate([*parts, -sum(parts)], axis=1).astype(np.float64)).to(DTYPES[dtype]).cuda()
    packed = torch.from_numpy(np.tile(rng.integers(0, 256, size=(whole, k // 16)).astype(np.uint8), (1, 8))).cuda()
    scales = torch.from_numpy(np.tile(2 ** rng.uniform(-6, 8, size=(whole, k // 8 // 32)), (1, 8))).to(DTYPES[dtype]).cuda()
    want = w4.matvec(x, w4.W4Weights(packed, scales))
    assert (want != 0).float().mean() > 0.2  # (there are rounding errors to compare)
    for _ in range(3):
        assert torch.equal(w4.matvec(x, w4.W4Weights(packed[:n].contiguous(), scales[:n].contiguous())), want[:, :n])


def test_results_over_inputs():
    """A product's rows are read until its end; the experts' are not, so a layer's output may take their place."""
    from deepep_amd import w4

    rng = np.random.default_rng(15)
    square = w4.W4Weights(*_weights(rng, (256, 256), 64, True, "bf16")[0])
    held = torch.randn((6, 256), device="cuda").bfloat16()
    x, before = held[:4], held.clone()
    for out in (x, held[1:5], held[2:]):
        with pytest.raises(ValueError):
            w4.matvec(x, square, out=out)
    assert torch.equal(held, before)
    assert torch.equal(w4.matvec(held[:3], square, out=held[3:]), w4.matvec(before[:3].clone(), square))
    gate_up, down = w4.W4Weights(*_weights(rng, (4, 128, 256), 64, False, "bf16")[0]), w4.W4Weights(*_weights(rng, (4, 256, 64), 64, False, "bf16")[0])
    x, ids, route_weights = torch.randn((5, 256), device="cuda").bfloat16(), torch.randint(-1, 4, (5, 2), device="cuda"), torch.rand((5, 2), device="cuda")
    want = w4.expert_ffn(x, ids, route_weights, gate_up, down)
    assert torch.equal(w4.expert_ffn(x, ids, route_weights, gate_up, down, out=x), want) and torch.equal(x, want)


@pytest.mark.parametrize("tokens,hidden,inter,topk,experts,group,zeros", [
    (1, 512, 128, 1, 2, 128, False), (4, 128, 128, 2, 4, 32, True), (3, 512, 320, 3, 8, 64, True), (8, 384, 256, 2, 4, 128, False),
    (2, 2048, 512, 2, 4, 128, True), (40, 256, 192, 2, 3, 64, False), (5, 768, 384, 2, 4, 384, True), (2, 7168, 256, 2, 4, 128, False),
])
def test_rows_between_the_products_keep_16_bits(tokens, hidden, inter, topk, experts, group, zeros):
    """FP16 results within six deviations of what the sums and 16 bits of mantissa may be off by, and half a last place.  (The oracle's test
    shows that rows of 8 bits leave this bound in many places.)"""
    from deepep_amd import w4

    rng = np.random.default_rng(hidden + inter)
    gate_up, gate_up_host = _weights(rng, (experts, 2 * inter, hidden), group, zeros, "fp16")
    down, down_host = _weights(rng, (experts, hidden, inter), group, zeros, "fp16")
    x, wide = _rows(rng, (tokens, hidden), "fp16")
    x = x * 0.25
    wide = x.double().cpu().numpy()
    ids, route_weights = np.argsort(rng.random((tokens, experts)), axis=1)[:, :topk], rng.random((tokens, topk)).astype(np.float32)
    y = w4.expert_ffn(x, torch.from_numpy(ids).cuda(), torch.from_numpy(route_weights).cuda(), w4.W4Weights(*gate_up), w4.W4Weights(*down))
    want, deviation = ow4.experts_and_deviation(wide, ids, route_weights.astype(np.float64), gate_up_host, down_host)
    off = np.abs(y.double().cpu().numpy() - want)
    bound = 6 * deviation + 2.0**-11 * np.abs(want) + 2.0**-25
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("rows,n,k,group,zeros,dtype", [
    (1, 64, 384, 384, False, "bf16"), (3, 40, 1152, 384, True, "fp16"), (2, 33, 1920, 640, False, "bf16"), (17, 48, 2688, 896, True, "bf16"),
    (5, 130, 16128, 384, False, "fp16"), (2, 20, 16128, 5376, True, "bf16"), (1, 16, 16000, 640, True, "bf16"),
])
def test_groups_that_are_no_power_of_two(rows, n, k, group, zeros, dtype):
    """Which of its row's groups a half unit belongs to is found with a rounded reciprocal."""
    test_matvec(rows, n, k, group, zeros, dtype)
