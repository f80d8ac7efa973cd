"""The 64-bit router oracle: hand-sized cases, its gradients against differences."""

import numpy as np
import pytest

from oracle import router as orouter


def test_choice_by_hand():
    z = np.array([1.0, 3.0, 3.0, -np.inf, 2.0])
    assert orouter.choose(z, 3) == [1, 2, 4]
    assert orouter.choose(z, 5) == [1, 2, 4, 0, -1]
    assert orouter.choose(z, 2, real=False) == [-1, -1]
    assert orouter.choose(np.array([0.0, np.nan, 5.0]), 2) == [1, 2]
    # the bias decides the choice
    assert orouter.choose(np.array([0.0, 0.0, 0.0]), 1, "sigmoid", bias=[0.0, 0.25, 0.0]) == [1]


def test_groups_by_hand():
    z = np.array([4.0, -9.0, 3.0, 2.9, 0.0, 0.0])
    assert orouter.choose(z, 2, groups=3, topk_groups=1) == [0, 1]  # the largest key
    assert orouter.choose(z, 2, "sigmoid", groups=3, topk_groups=1) == [2, 3]  # the sum of two
    assert orouter.choose(np.array([-np.inf, -np.inf, 1.0, -np.inf]), 2, "sigmoid", groups=2, topk_groups=1) == [2, -1]


def test_weights_by_hand():
    z = np.log(np.array([1.0, 2.0, 5.0]))
    np.testing.assert_allclose(orouter.weights_of(z, [2, 1], normalize=True), [5 / 7, 2 / 7])
    np.testing.assert_allclose(orouter.weights_of(z, [2, -1], normalize=False, scale=2.0), [1.25, 0.0])
    np.testing.assert_allclose(orouter.weights_of(np.zeros(3), [0, 2], "sigmoid"), [0.5, 0.5])


def test_balance_by_hand():
    # two tokens, both to expert 0, probabilities (3/4, 1/4): f = (2, 0), P = (3/4, 1/4)
    z = np.log(np.array([[3.0, 1.0], [3.0, 1.0], [1.0, 1.0]]))
    losses, counts, members = orouter.balance(z, [[0], [0], [-1]])
    np.testing.assert_allclose(losses, [1.5])
    assert counts.tolist() == [[2, 0]] and members.tolist() == [2]
    losses, counts, members = orouter.balance(z, [[0], [1], [-1]], offsets=[0, 1, 1, 3])
    np.testing.assert_allclose(losses, [1.5, 0.0, 0.5])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_gradients_against_differences(score, normalize):
    rng = np.random.default_rng(5)
    z = rng.normal(size=(6, 7))
    z[:, 3] = -np.inf
    ids = [orouter.choose(row, 3, score) for row in z]
    ids[2] = [-1, -1, -1]
    g = rng.normal(size=(6, 3))
    g_losses = rng.normal(size=(2,))
    offsets = [0, 4, 6]

    def total(z):
        value = sum((g[t] * orouter.weights_of(z[t], ids[t], score, normalize, 1.5)).sum() for t in range(6))
        return value, (orouter.balance(z, ids, score, offsets)[0] * g_losses).sum()

    exact = np.stack([orouter.weights_gradient(z[t], ids[t], g[t], score, normalize, 1.5) for t in range(6)])
    exact_balance = orouter.balance_gradient(z, ids, g_losses, score, offsets)
    for t in range(6):
        for e in range(7):
            if e == 3:
                assert exact[t, e] == 0 and exact_balance[t, e] == 0
                continue
            step = np.zeros_like(z)
            step[t, e] = 1e-5
            (a, c), (b, d) = total(z + step), total(z - step)
            assert abs((a - b) / 2e-5 - exact[t, e]) < 1e-8
            assert abs((c - d) / 2e-5 - exact_balance[t, e]) < 1e-8
