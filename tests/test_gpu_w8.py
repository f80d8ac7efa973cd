"""Products in 8-bit integers on the GPU: integer sums exactly, scaled in 32 bits and rounded once."""

import numpy as np
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _codes(rng, *shape):
    return torch.from_numpy(rng.integers(-127, 128, size=shape).astype(np.int8)).cuda()


def _make(rows, n, k):
    rng = np.random.default_rng(rows * 31 + n * 7 + k)
    scales = lambda count: torch.from_numpy((0.5 + rng.random(count)).astype(np.float32) * 0.01).cuda()  # noqa: E731
    return (_codes(rng, rows, k), scales(rows)), (_codes(rng, n, k), scales(n))


def _want(x, w):
    """The exact value, and in it the sums as integers."""
    sums = x[0].cpu().numpy().astype(np.int64) @ w[0].cpu().numpy().astype(np.int64).T
    return sums * x[1].double().cpu().numpy()[:, None] * w[1].double().cpu().numpy()


SIZES = [  # rows, n, k
    (1, 1, 16), (1, 4096, 7168), (1, 33, 48), (2, 17, 64), (3, 100, 2880), (4, 257, 128), (7, 40, 4112), (8, 64, 1024), (15, 1407, 208), (16, 256, 512), (17, 96, 8192), (31, 65, 80), (32, 128, 96),
    (33, 1407, 2880), (64, 300, 640), (65, 64, 272), (100, 129, 1040), (128, 256, 256), (129, 255, 144), (200, 513, 512), (256, 256, 1024), (257, 259, 272), (300, 1, 4096), (600, 130, 336),
    (1025, 72, 128), (5, 24, 65536), (300, 40, 16384),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_codes(rows, n, k, dtype):
    from deepep_amd import w8

    x, w = _make(rows, n, k)
    y = w8.matmul(x, w8.W8Weights(*w), dtype=DTYPES[dtype])
    assert y.dtype == DTYPES[dtype] and y.shape == (rows, n)
    want = _want(x, w)
    # the sum as a 32-bit number and two products of it: three roundings, then the result's
    bound = 4 * od.EPS32 * np.abs(want)
    off = np.abs(y.double().cpu().numpy() - want)
    bound = bound + od.HALF[dtype] * (np.abs(want) + bound) + od.TINY[dtype]
    assert (off <= bound).all(), np.argwhere(off > bound)[:5].tolist()
    assert torch.equal(y, w8.matmul(x, w8.W8Weights(*w), dtype=DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 7168), (3, 48), (5, 2880), (70, 2064), (2, 65536)])
def test_tokens(rows, k, dtype):
    from deepep_amd import w8

    rng = np.random.default_rng(rows + k)
    x = torch.from_numpy(rng.normal(size=(rows, k)) * (0.1 + rng.random((rows, 1)))).to(DTYPES[dtype]).cuda()
    if rows > 1:
        x[1] = 0
    codes, scales = w8.quantize_tokens(x)
    target, want = od.tokens(x.double().cpu().numpy())
    assert (np.abs(scales.double().cpu().numpy() - want) <= 2 * od.EPS32 * want).all()
    assert (np.abs(codes.double().cpu().numpy() - target) <= 0.5 + 8 * od.EPS32 * 127).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 512), (300, 512), (300, 528), (2, 2064), (257, 2048), (257, 4112), (300, 8192), (300, 8208), (3, 16384), (260, 16384), (3, 16400), (300, 20000)])
def test_tokens_of_all_widths(rows, k, dtype):
    """Rows in a workgroup's registers, in each number of pieces, and rows that do not fit."""
    from deepep_amd import w8

    rng = np.random.default_rng(rows * 7 + k)
    x = torch.from_numpy(rng.normal(size=(rows, k)) * (0.1 + rng.random((rows, 1)))).to(DTYPES[dtype]).cuda()
    x[-1, -1] = 7.5  # a row's largest value in its last place
    codes, scales = w8.quantize_tokens(x)
    target, want = od.tokens(x.double().cpu().numpy())
    assert (np.abs(scales.double().cpu().numpy() - want) <= 2 * od.EPS32 * want).all()
    assert (np.abs(codes.double().cpu().numpy() - target) <= 0.5 + 8 * od.EPS32 * 127).all()
    assert codes[-1, -1] == 127


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_wide_rows_are_quantised_in_the_call(rows):
    from deepep_amd import w8

    rng = np.random.default_rng(rows)
    x = torch.from_numpy(rng.normal(size=(rows, 528))).bfloat16().cuda()
    _, w = _make(1, 77, 528)
    weights = w8.W8Weights(*w)
    y = w8.matmul(x, weights)
    assert y.dtype == torch.bfloat16 and torch.equal(y, w8.matmul(w8.quantize_tokens(x), weights))
    assert torch.equal(w8.matmul(list(w8.quantize_tokens(x)), weights), y)
    assert w8.matmul(x, weights, dtype=torch.float32).dtype == torch.float32


def test_largest_sums_do_not_pass_31_bits():
    from deepep_amd import w8

    k = 65536
    for sign in (1, -1):
        x = torch.full((20, k), 127, dtype=torch.int8, device="cuda")
        w = torch.full((3, k), 127 * sign, dtype=torch.int8, device="cuda")
        one = torch.ones(20, device="cuda")
        y = w8.matmul((x, one), w8.W8Weights(w, torch.ones(3, device="cuda")), dtype=torch.float32)
        assert (y == float(np.float32(127 * 127 * k * sign))).all()
    x = torch.full((1, k), -128, dtype=torch.int8, device="cuda")
    y = w8.matmul((x, torch.ones(1, device="cuda")), w8.W8Weights(x.clone(), torch.ones(1, device="cuda")), dtype=torch.float32)
    assert y.item() == 128.0 * 128 * k


def test_rows_that_are_not_finite():
    from deepep_amd import w8

    x = torch.ones(3, 64, dtype=torch.bfloat16, device="cuda")
    x[1, 5] = float("nan")
    x[2, 5] = float("inf")
    w = w8.W8Weights(torch.ones(8, 64, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda"))
    y = w8.matmul(x, w)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", [64, 2064, 20000])
def test_infinities_keep_their_sign(dtype, k):
    from deepep_amd import w8

    most = torch.finfo(DTYPES[dtype]).max
    x = torch.full((4, k), most, dtype=DTYPES[dtype], device="cuda")
    x[0, 5], x[1, k - 1], x[2, 5], x[2, 6] = float("inf"), -float("inf"), float("inf"), -float("inf")
    x[3, 5] = float("nan")
    codes, scales = w8.quantize_tokens(x)
    want = torch.zeros(3, k, dtype=torch.int8)
    want[0, 5], want[1, k - 1], want[2, 5], want[2, 6] = 127, -127, 127, -127
    assert torch.equal(codes[:3].cpu(), want) and (scales[:3] == float("inf")).all() and torch.isnan(scales[3])
    y = w8.matmul((codes, scales), w8.W8Weights(torch.ones(8, k, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")))
    assert (y[0] == float("inf")).all() and (y[1] == -float("inf")).all() and torch.isnan(y[2:]).all()


def test_no_rows():
    from deepep_amd import w8

    x, w = _make(1, 5, 32)
    y = w8.matmul((x[0][:0], x[1][:0]), w8.W8Weights(*w))
    assert y.shape == (0, 5)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_captured_products_replay(rows):
    from deepep_amd import w8

    rng = np.random.default_rng(rows)
    x = torch.from_numpy(rng.normal(size=(rows, 1040))).bfloat16().cuda()
    _, w = _make(1, 130, 1040)
    weights = w8.W8Weights(*w)
    w8.matmul(x, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = w8.matmul(x, weights)
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.normal(size=(rows, 1040))))
        want = w8.matmul(x, weights)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_two_streams_at_once():
    """k in parts, whose sums are scratch of each call, and rows quantised in the call."""
    from deepep_amd import ops, w8

    assert ops.product_choices("w8", 300, 40, 16384)[0]["parts"] > 1
    gen = torch.Generator().manual_seed(4)
    rows = [torch.randn(300, 16384, generator=gen).bfloat16().cuda() for _ in range(2)]
    weights = w8.W8Weights(*_make(1, 40, 16384)[1])
    want = [w8.matmul(x, weights) for x in rows]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in rows], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(w8.matmul(rows[i], weights))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_matrix_quantised_once():
    from deepep_amd import w8

    gen = torch.Generator().manual_seed(0)
    matrix, x = torch.randn(96, 512, generator=gen).cuda() * 0.05, torch.randn(9, 512, generator=gen).cuda().bfloat16()
    y = w8.matmul(x, w8.quantize(matrix), dtype=torch.float32)
    want = x.float() @ matrix.T
    # each side is off by at most half a step of 127 to its largest value, about 3.5 of its deviations: sqrt(2) * 3.5 / 127 / sqrt(12) of the result
    assert ((y - want).norm() / want.norm()).item() < 0.016
