"""The feed-forward block and the 8-bit products at sizes for the ways of making a product that the other modules' sizes do not reach: streams of many workgroups, tiles of 256 and pairs with k in
parts, the backward's products apart.  ``tests/test_product_choice.py`` checks that all modules' sizes together leave none out."""

import pytest

from tests import test_gpu_dense_ways as ways

pytestmark = pytest.mark.gpu

SIZES = [  # tokens, hidden, inter
    (5, 80, 4496), (3, 4104, 8200), (10, 9936, 72),  # streams of more than 512 groups of columns
    (77, 1544, 1304), (67, 8, 4392),  # pairs, k in parts: gate and up; down
    (2360, 8936, 896), (2476, 7672, 1928), (7078, 584, 7296),  # tiles of 256, k in parts: gate and up; dh; down
    (8460, 400, 912), (7235, 136, 1512), (2500, 264, 136),  # the backward's three together, of 256 and of 128, k in parts
    (1682, 3608, 904), (16226, 192, 1400), (14714, 240, 3104),  # apart, k whole: pairs and ring
    (14249, 56, 1752), (18852, 328, 2184), (3078, 624, 5832), (3511, 960, 8112), (14685, 392, 3680),  # apart, k in parts: ring, pairs, tiles of 256
]
CODES = [(3, 8360, 176), (1, 33000, 4096), (65, 3, 7776), (140, 4500, 7184), (5582, 727, 18688)]  # rows, n, k


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
def test_block(tokens, hidden, inter, dtype):
    ways.test_block(tokens, hidden, inter, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", CODES)
def test_codes(rows, n, k, dtype):
    ways.test_codes(rows, n, k, dtype)
