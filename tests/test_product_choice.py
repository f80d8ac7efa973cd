"""How the gated block's and the 8-bit products are cut up (host arithmetic, no GPU needed)."""

import ctypes
import math
import random

import pytest

from deepep_amd import _lib, ops
from tests import test_gpu_dense, test_gpu_dense_choices, test_gpu_dense_ways, test_gpu_w8

MOST_WORKGROUPS = 0x7FFFFF  # of 512 threads


@pytest.mark.parametrize("operation,sizes", [
    ("ffn", (2097151, 8, 32768)), ("ffn", (2097151, 8, 65536)), ("ffn", (2097151, 65536, 8)), ("ffn", (2097151, 65536, 65536)), ("ffn", (1, 65536, 65536)),
    ("ffn_backward", (2097151, 8, 65536)), ("ffn_backward", (2097151, 65536, 8)), ("ffn_backward", (2097151, 65536, 65536)),
    ("w8", (2097151, 131072, 16)), ("w8", (2097151, 131072, 65536)), ("w8", (1, 2097151, 65536)), ("w8", (261888, 2097151, 16)),
])
def test_cuts_of_the_largest_sizes_can_be_launched(operation, sizes):
    choices = ops.product_choices(operation, *sizes)
    together = [c for c in choices if c["together"]]
    assert all(c["workgroups"] <= MOST_WORKGROUPS for c in choices) and sum(c["workgroups"] for c in together) <= MOST_WORKGROUPS


@pytest.mark.parametrize("operation,sizes,ways", [
    # few rows on large matrices: nothing but the reading of the matrix counts
    ("ffn", (1, 8192, 28672), ["stream", "stream"]), ("ffn", (4, 7168, 18432), ["stream", "stream"]), ("w8", (1, 128256, 4096), ["stream"]), ("w8", (4, 8192, 28672), ["stream"]),
    # and many short workgroups their own starts
    ("w8", (6, 62901, 432), ["pairs"]), ("ffn", (6, 264, 28176), ["pairs", "stream"]),
    # what the rules were measured at before
    ("ffn", (1, 7168, 2048), ["stream", "stream"]), ("ffn", (33, 2880, 1408), ["stream", "stream"]), ("ffn", (512, 7168, 2048), ["ring", "ring"]),
    ("ffn", (8192, 7168, 2048), ["large", "large"]), ("ffn_backward", (8192, 7168, 2048), ["large"] * 4), ("ffn_backward", (1000, 2880, 1408), ["ring", "pairs", "pairs", "pairs"]),
    ("w8", (1, 4096, 7168), ["stream"]), ("w8", (100, 1407, 2880), ["stream"]), ("w8", (8192, 4096, 7168), ["large"]),
])
def test_ways_of_known_sizes(operation, sizes, ways):
    assert [c["way"] for c in ops.product_choices(operation, *sizes)] == ways


def test_products_that_cannot_be_launched_are_refused():
    lib, at = _lib.load(), 1 << 20  # (no call below reaches memory)
    w = ops._W8(at, at, 2097151, 16)
    assert lib.dpep_w8_matmul(ctypes.byref(w), at, at, 2097151, 1, at, at, None) == -1
    assert "too large" in lib.dpep_last_error().decode()
    assert lib.dpep_w8_matmul_scratch_bytes(2097151, 2097151, 16) == 0


def test_sizes_that_no_call_takes():
    lib = _lib.load()
    for bad in (("ffn", 1, 12, 8), ("ffn", 1, 8, 65544), ("ffn_backward", -1, 8, 8), ("ffn", 1 << 21, 8, 8), ("w8", 1, 0, 16), ("w8", 1, 8, 24), ("w8", 1 << 21, 8, 16)):
        with pytest.raises(ValueError, match="product_choices"):
            ops.product_choices(*bad)
    assert lib.dpep_product_choices(0, 1, 8, 8, None) == -1 and lib.dpep_product_choices(3, 1, 8, 8, ctypes.byref((ops._ProductChoice * 4)())) == -1
    for bad in ((-1, 8, 8), (1 << 21, 8, 8), (1, 1 << 30, 8), (1, 8, 0x7FFFFFF8)):
        assert lib.dpep_gated_ffn_scratch_bytes(*bad) == 0 and lib.dpep_gated_ffn_backward_scratch_bytes(*bad) == 0
    for bad in ((-1, 8, 16), (1, 1 << 30, 16), (1, 8, 0x7FFFFFF0)):
        assert lib.dpep_w8_matmul_scratch_bytes(*bad) == 0


_PRODUCTS = {"ffn": ("gate and up", "down"), "ffn_backward": ("dh", "dx", "dw", "dw"), "w8": ("codes",)}


def _made(operation, sizes):
    """What of the kernels a call takes: which product, way, shape of its stream, k whole or in parts, alone or with the two others."""
    return {(product, c["way"], c["stream"], c["parts"] > 1, c["together"]) for product, c in zip(_PRODUCTS[operation], ops.product_choices(operation, *sizes))}


def _parameters(test, names):
    return next(mark.args[1] for mark in test.pytestmark if mark.name == "parametrize" and mark.args[0] == names)


def test_the_gpu_tests_sizes_take_every_way_there_is():
    blocks = (test_gpu_dense.SIZES + _parameters(test_gpu_dense.test_many_tokens, "tokens,hidden,inter") + test_gpu_dense_ways.SIZES + test_gpu_dense_choices.SIZES)
    codes = test_gpu_w8.SIZES + _parameters(test_gpu_dense_ways.test_codes, "rows,n,k") + test_gpu_dense_choices.CODES
    tested = set().union(*(_made(operation, sizes) for sizes in blocks for operation in ("ffn", "ffn_backward")), *(_made("w8", sizes) for sizes in codes))
    rng, reached = random.Random(3), {}
    log = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))  # noqa: E731
    for _ in range(60000):
        operation = rng.choice(sorted(_PRODUCTS))
        sizes = (log(1, 20000), log(1, 200000), log(1, 4096) * 16) if operation == "w8" else (log(1, 20000), log(1, 3600) * 8, log(1, 3600) * 8)
        if sizes[1] * sizes[2] < 1.5e9 and sizes[0] * max(sizes[1:]) < 1e9:
            for made in _made(operation, sizes):
                reached.setdefault(made, (operation, sizes))
    assert len(reached) > 50
    assert not {made: sizes for made, sizes in reached.items() if made not in tested}
