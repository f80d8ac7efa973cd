"""The 64-bit oracle of norm and gated block: gradients against central differences, quantisers against the types' own rounding."""

import numpy as np
import pytest
import torch

from oracle import dense as od


def _difference(f, at, step=1e-6):
    """Gradient of f at an array by central differences."""
    grad = np.zeros_like(at)
    for i in np.ndindex(*at.shape):
        keep = at[i]
        at[i] = keep + step
        up = f()
        at[i] = keep - step
        down = f()
        at[i] = keep
        grad[i] = (up - down) / (2 * step)
    return grad


def test_norm_gradient_matches_differences():
    rng = np.random.default_rng(0)
    s, w, g, more = rng.normal(size=(3, 16)), rng.normal(size=16), rng.normal(size=(3, 16)), rng.normal(size=(3, 16))
    grad, _, grad_w, _ = od.norm_backward(g, s, w, 1e-3, more)
    loss = lambda: (od.norm(s, w, 1e-3)[0] * g).sum() + (s * more).sum()  # noqa: E731
    np.testing.assert_allclose(grad, _difference(loss, s), rtol=1e-6, atol=1e-8)
    np.testing.assert_allclose(grad_w, _difference(loss, w), rtol=1e-6, atol=1e-8)


def test_ffn_gradients_match_differences():
    rng = np.random.default_rng(1)
    x, gate_up, down, g = rng.normal(size=(3, 8)), rng.normal(size=(16, 8)), rng.normal(size=(8, 8)), rng.normal(size=(3, 8))
    loss = lambda: (od.ffn(x, gate_up, down, "fp32")["y"] * g).sum()  # noqa: E731
    for (grad, _), at in zip(od.ffn_backward(g, x, gate_up, down, "fp32"), (x, gate_up, down)):
        np.testing.assert_allclose(grad, _difference(loss, at), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ffn_bounds_hold_for_torch_products_in_32_bits(dtype):
    torch_type = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    gen = torch.Generator().manual_seed(2)
    x, gate_up, down = (torch.randn(s, generator=gen).to(torch_type) for s in ((5, 64), (80, 64), (64, 40)))
    g, u = (x.float() @ gate_up.float().T).chunk(2, dim=1)
    y = ((g * torch.sigmoid(g) * u).to(torch_type).float() @ down.float().T).to(torch_type)
    want = od.ffn(*(t.double().numpy() for t in (x, gate_up, down)), dtype)
    off = np.abs(y.double().numpy() - want["y"])
    assert (off <= want["y_off"]).all()
    assert (want["y_off"] <= 0.5 * np.abs(want["y"]).max()).all()  # and says something


def test_e4m3_bound_is_half_a_step():
    values = torch.linspace(-448, 448, 20001, dtype=torch.float64)
    rounded = values.float().to(torch.float8_e4m3fn).double()
    off = (rounded - values).abs().numpy()
    assert (off <= od.e4m3_bound(values.numpy()) * (1 + 1e-6)).all()
    small = torch.linspace(-0.02, 0.02, 4001, dtype=torch.float64)
    assert ((small.float().to(torch.float8_e4m3fn).double() - small).abs().numpy() <= od.e4m3_bound(small.numpy()) * (1 + 1e-6)).all()
