"""The 64-bit oracle of the 4-bit products: by hand, and that its deviation tells 16 bits of mantissa between the two expert products
from 8."""

import numpy as np
import pytest

from oracle import w4 as ow4


def test_product_by_hand():
    packed = np.array([[0x98, 0x0F]], dtype=np.uint8)  # codes 8, 9, 15, 0
    x = np.array([[1.0, 2.0, 3.0, 4.0]])
    assert ow4.product(x, (packed, np.array([[0.5]]), None))[0].tolist() == [[0.5 * (0 + 2 + 21 - 32)]]
    assert ow4.product(x, (packed, np.array([[0.5]]), np.array([[9]])))[0].tolist() == [[0.5 * (-1 + 0 + 18 - 36)]]


def test_bf16_rounds_to_nearest_even():
    assert ow4.bf16([1.0, 1 + 2.0**-8, 1 + 3 * 2.0**-8, 1 + 2.0**-8 + 2.0**-20, -(1 + 2.0**-9)]).tolist() == [1.0, 1.0, 1 + 2.0**-6, 1 + 2.0**-7, -1.0]


@pytest.mark.parametrize("tokens,hidden,inter,topk,experts,group,zeros", [
    (4, 128, 128, 1, 4, 32, True), (3, 512, 320, 3, 8, 64, True), (8, 384, 256, 2, 4, 128, False), (2, 2048, 512, 2, 4, 128, False),
])
def test_deviation_finds_rows_of_8_bits(tokens, hidden, inter, topk, experts, group, zeros):
    """FP16 results, as the GPU's are tested: rows held as pairs of BF16 stay within six deviations and a rounding, rows held as one
    BF16 leave that bound in many places."""
    rng = np.random.default_rng(hidden)

    def weights(*shape):
        scales = (0.02 * (0.25 + rng.random((*shape[:-1], shape[-1] // group)))).astype(np.float16).astype(np.float64)
        return (rng.integers(0, 256, size=(*shape[:-1], shape[-1] // 2)).astype(np.uint8), scales, rng.integers(0, 16, size=scales.shape) if zeros else None)

    gate_up, down = weights(experts, 2 * inter, hidden), weights(experts, hidden, inter)
    x = 0.25 * rng.normal(size=(tokens, hidden)).astype(np.float16).astype(np.float64)
    ids, route_weights = np.argsort(rng.random((tokens, experts)), axis=1)[:, :topk], rng.random((tokens, topk))
    want, deviation = ow4.experts_and_deviation(x, ids, route_weights, gate_up, down)
    np.testing.assert_allclose(want, ow4.experts(x, ids, route_weights, gate_up, down)[0], rtol=1e-9, atol=1e-12)
    bound = 6 * deviation + 2.0**-11 * np.abs(want) + 2.0**-25

    def outside(hold):
        got = ow4.experts_and_deviation(x, ids, route_weights, gate_up, down, hold)[0].astype(np.float16).astype(np.float64)
        return (np.abs(got - want) > bound).mean()

    assert outside(lambda h: ow4.bf16(h) + ow4.bf16(h - ow4.bf16(h))) == 0
    assert outside(ow4.bf16) > 0.2
