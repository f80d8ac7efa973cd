"""The root-mean-square norm, its 8-bit outputs and its gradients on the GPU against the 64-bit oracle, within half a step of the output's
type and the oracle's bound on 32-bit sums."""

import numpy as np
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _rows(rng, tokens, hidden, dtype, scale=1.0):
    x = rng.normal(size=(tokens, hidden)) * scale * (0.25 + rng.random((tokens, 1)))
    return torch.from_numpy(x).to(DTYPES[dtype]).cuda()


def _weight(rng, hidden, dtype):
    return torch.from_numpy(1.0 + 0.3 * rng.normal(size=hidden)).to(DTYPES[dtype]).cuda()


def _wide(t):
    return None if t is None else t.double().cpu().numpy()


def _check(got, want, bound, dtype):
    off = np.abs(_wide(got) - want)
    bound = bound + od.HALF[dtype] * (np.abs(want) + bound) + od.TINY[dtype]
    assert (off <= bound).all(), float((off / np.maximum(bound, 1e-300)).max())


SIZES = [  # tokens, hidden, x, weight, residual
    (1, 8, "bf16", "bf16", False), (1, 7168, "bf16", "bf16", True), (3, 64, "fp16", "fp32", True), (5, 512, "bf16", "fp32", False), (5, 520, "fp16", "fp16", True),
    (2, 1000, "fp32", "fp32", True), (7, 2048, "bf16", "bf16", True), (4, 2056, "bf16", "fp32", True), (3, 2880, "fp16", "fp16", False), (2, 4104, "fp32", "fp32", False),
    (9, 5120, "bf16", "bf16", True), (2, 8192, "bf16", "bf16", False), (2, 8200, "fp16", "fp32", True), (3, 16384, "bf16", "bf16", True), (130, 256, "fp32", "fp32", True),
    (1025, 72, "bf16", "fp32", True), (600, 2880, "bf16", "bf16", True),
]


def _make(tokens, hidden, dtype, weight, residual, seed=0):
    rng = np.random.default_rng(tokens * 100003 + hidden + seed)
    return _rows(rng, tokens, hidden, dtype, 3.0), _weight(rng, hidden, weight), _rows(rng, tokens, hidden, dtype) if residual else None, rng


@pytest.mark.parametrize("tokens,hidden,dtype,weight,residual", SIZES)
def test_norm(tokens, hidden, dtype, weight, residual):
    from deepep_amd import dense

    x, w, r, _ = _make(tokens, hidden, dtype, weight, residual)
    got = dense.rms_norm(x, w, r, eps=EPS)
    assert got.y.dtype == x.dtype and got.codes is None and got.scales is None
    if residual:
        assert torch.equal(got.stream, (x.float() + r.float()).to(x.dtype))
    else:
        assert got.stream is x
    v, rstd = od.norm(_wide(got.stream), _wide(w), EPS)
    _check(got.rstd, rstd, od.NORM_SLACK * rstd, "fp32")
    _check(got.y, v, od.NORM_SLACK * np.abs(v), dtype)
    again = dense.rms_norm(x, w, r, eps=EPS)
    assert torch.equal(got.y, again.y) and torch.equal(got.rstd, again.rstd)


@pytest.mark.parametrize("quantize,unit", [("fp8", 16), ("mxfp8", 32), ("int8", 16)])
@pytest.mark.parametrize("tokens,hidden,dtype,weight,residual", [s for s in SIZES if s[1] % 16 == 0] + [(3, 144, "bf16", "bf16", True), (2, 48, "fp16", "fp32", False)])
def test_eight_bits(tokens, hidden, dtype, weight, residual, quantize, unit):
    from deepep_amd import dense

    if hidden % unit:
        pytest.skip("not a multiple of the format's unit")
    x, w, r, _ = _make(tokens, hidden, dtype, weight, residual)
    if tokens > 2:
        x[1] = 0
        if r is not None:
            r[1] = 0
    got = dense.rms_norm(x, w, r, eps=EPS, quantize=quantize)
    plain = dense.rms_norm(x, w, r, eps=EPS)
    assert torch.equal(got.y, plain.y) and torch.equal(got.stream, plain.stream)
    without = dense.rms_norm(x, w, r, eps=EPS, quantize=quantize, output=False)
    assert without.y is None and torch.equal(without.scales, got.scales) and torch.equal(without.codes.view(torch.uint8), got.codes.view(torch.uint8))
    v, _ = od.norm(_wide(got.stream), _wide(w), EPS)
    slack = 2 * od.NORM_SLACK
    if quantize == "fp8":
        target, scales = od.fp8_blocks(v)
        _check(got.scales, scales, slack * scales, "fp32")
        assert (np.abs(_wide(got.codes.float()) - target) <= od.e4m3_bound(target) * (1 + 1e-9) + slack * np.abs(target)).all()
    elif quantize == "int8":
        target, scales = od.tokens(v)
        _check(got.scales, scales, slack * scales, "fp32")
        assert (np.abs(_wide(got.codes) - target) <= 0.5 + slack * 127).all()
        assert int(got.codes.min()) >= -127
    else:
        blocks = v.reshape(tokens, hidden // 32, 32)
        largest = np.maximum(np.abs(blocks).max(axis=2), 2.0**-119)
        low, high = (np.floor(np.log2(largest * f)) + 127 - 8 for f in (1 - slack, 1 + slack))
        byte = got.scales.cpu().numpy().astype(np.float64)
        assert ((byte == low) | (byte == high)).all()
        target = np.clip(blocks * 2.0 ** (127 - byte[:, :, None]), -448, 448).reshape(tokens, hidden)
        assert (np.abs(_wide(got.codes.float()) - target) <= od.e4m3_bound(target) * (1 + 1e-9) + slack * np.abs(target)).all()


def test_codes_are_those_of_the_casts_where_the_norm_changes_nothing():
    """Rows of +-1 with weights that are powers of two: v needs no rounding, so y and v are the same and the codes are per_token_cast_to_fp8's, mx_quant's and
    quantize_tokens' bit for bit."""
    from deepep_amd import dense, ops, w8
    from deepep_amd.utils import per_token_cast_to_fp8

    gen = torch.Generator().manual_seed(3)
    x = (torch.randint(0, 2, (6, 640), generator=gen) * 2 - 1).bfloat16().cuda()
    w = torch.exp2(torch.randint(-3, 4, (640,), generator=gen).float()).bfloat16().cuda()
    y = (x.float() * w.float()).bfloat16()
    for quantize, cast in (("fp8", per_token_cast_to_fp8), ("mxfp8", ops.mx_quant), ("int8", w8.quantize_tokens)):
        got = dense.rms_norm(x, w, eps=0.0, quantize=quantize)
        assert torch.equal(got.y, y)
        codes, scales = cast(y)
        assert torch.equal(got.codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(got.scales, scales)


@pytest.mark.parametrize("tokens,hidden,dtype,weight,residual", SIZES)
def test_gradients(tokens, hidden, dtype, weight, residual):
    from deepep_amd import dense

    x, w, r, rng = _make(tokens, hidden, dtype, weight, residual)
    normed = dense.rms_norm(x, w, r, eps=EPS)
    g = _rows(rng, tokens, hidden, dtype)
    more = _rows(rng, tokens, hidden, dtype) if residual else None
    grad_x, grad_w = dense.rms_norm_backward(g, normed.stream, w, normed.rstd, more)
    assert grad_x.dtype == x.dtype and grad_w.dtype == torch.float32
    want, bound, want_w, bound_w = od.norm_backward(_wide(g), _wide(normed.stream), _wide(w), EPS, _wide(more))
    _check(grad_x, want, bound, dtype)
    _check(grad_w, want_w, bound_w, "fp32")
    again = dense.rms_norm_backward(g, normed.stream, w, normed.rstd, more)
    assert torch.equal(grad_x, again[0]) and torch.equal(grad_w, again[1])


@pytest.mark.parametrize("tokens,hidden,dtype", [(1300, 2056, "bf16"), (2050, 2880, "fp16"), (2100, 264, "bf16"), (4100, 4096, "bf16"), (4099, 1024, "fp32"), (9001, 512, "bf16"), (20000, 72, "fp16")])
def test_gradients_of_many_rows(tokens, hidden, dtype):
    """Sizes that take more workgroups than compute units, with all numbers of rows to one."""
    from deepep_amd import dense

    x, w, _, rng = _make(tokens, hidden, dtype, "fp32", False)
    normed = dense.rms_norm(x, w, eps=EPS)
    g = _rows(rng, tokens, hidden, dtype)
    grad_x, grad_w = dense.rms_norm_backward(g, normed.stream, w, normed.rstd)
    want, bound, want_w, bound_w = od.norm_backward(_wide(g), _wide(x), _wide(w), EPS)
    _check(grad_x, want, bound, dtype)
    _check(grad_w, want_w, bound_w, "fp32")
    again = dense.rms_norm_backward(g, normed.stream, w, normed.rstd)
    assert torch.equal(grad_x, again[0]) and torch.equal(grad_w, again[1])


@pytest.mark.parametrize("tokens,hidden,dtype,weight,residual", [
    (300, 1000, "bf16", "fp32", True), (257, 2048, "fp32", "fp32", False), (300, 5024, "fp16", "fp16", True), (260, 8192, "fp32", "fp32", True), (300, 8208, "bf16", "bf16", False),
    (257, 12320, "fp16", "fp32", True), (258, 16384, "bf16", "fp32", True), (257, 16384, "fp32", "fp32", False)])
def test_many_rows_of_all_widths(tokens, hidden, dtype, weight, residual):
    """More rows than compute units, in each number of pieces a thread: the norm, its codes and its gradients."""
    from deepep_amd import dense

    x, w, r, rng = _make(tokens, hidden, dtype, weight, residual)
    got = dense.rms_norm(x, w, r, eps=EPS)
    v, rstd = od.norm(_wide(got.stream), _wide(w), EPS)
    _check(got.rstd, rstd, od.NORM_SLACK * rstd, "fp32")
    _check(got.y, v, od.NORM_SLACK * np.abs(v), dtype)
    slack = 2 * od.NORM_SLACK
    if hidden % 16 == 0:
        coded = dense.rms_norm(x, w, r, eps=EPS, quantize="fp8")
        assert torch.equal(coded.y, got.y)
        target, scales = od.fp8_blocks(v)
        _check(coded.scales, scales, slack * scales, "fp32")
        assert (np.abs(_wide(coded.codes.float()) - target) <= od.e4m3_bound(target) * (1 + 1e-9) + slack * np.abs(target)).all()
        coded = dense.rms_norm(x, w, r, eps=EPS, quantize="int8", output=False)
        target, scales = od.tokens(v)
        _check(coded.scales, scales, slack * scales, "fp32")
        assert (np.abs(_wide(coded.codes) - target) <= 0.5 + slack * 127).all()
    g = _rows(rng, tokens, hidden, dtype)
    grad_x, grad_w = dense.rms_norm_backward(g, got.stream, w, got.rstd)
    want, bound, want_w, bound_w = od.norm_backward(_wide(g), _wide(got.stream), _wide(w), EPS)
    _check(grad_x, want, bound, dtype)
    _check(grad_w, want_w, bound_w, "fp32")


def test_no_rows():
    from deepep_amd import dense, w8

    x, w = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    got = dense.rms_norm(x, w, x.clone(), quantize="fp8")
    assert got.y.shape == (0, 64) and got.codes.shape == (0, 64) and got.scales.shape == (0, 1) and got.rstd.shape == (0,)
    grad_x, grad_w = dense.rms_norm_backward(x, x, w, got.rstd)
    assert grad_x.shape == (0, 64) and torch.equal(grad_w, torch.zeros(64, device="cuda"))
    codes, scales = w8.quantize_tokens(x)
    assert codes.shape == (0, 64) and scales.shape == (0,)


def test_rows_that_are_not_finite_stay_in_their_rows():
    from deepep_amd import dense

    rng = np.random.default_rng(5)
    x, w = _rows(rng, 4, 256, "bf16"), _weight(rng, 256, "bf16")
    clean = {q: dense.rms_norm(x, w, quantize=q) for q in ("fp8", "int8")}
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    for q, want in clean.items():
        got = dense.rms_norm(x, w, quantize=q)
        for row in (0, 3):
            assert torch.equal(got.y[row], want.y[row]) and torch.equal(got.codes[row].view(torch.uint8), want.codes[row].view(torch.uint8))
            assert torch.equal(got.scales[row], want.scales[row])
        assert torch.isnan(got.y[1]).all() and torch.isnan(got.scales[1]).all()
        assert torch.isnan(got.y[2, 9]) and not torch.isfinite(got.scales[2]).all()


def test_squares_that_pass_the_range_of_32_bits():
    """As documented: a row whose squares' sum overflows is normed to zeros with rstd 0, and no other row knows of it."""
    from deepep_amd import dense

    rng = np.random.default_rng(16)
    x, w = _rows(rng, 3, 256, "fp32"), _weight(rng, 256, "fp32")
    want = dense.rms_norm(x, w)
    x[1] = 1e20
    got = dense.rms_norm(x, w)
    assert got.rstd[1] == 0 and not got.y[1].any()
    for row in (0, 2):
        assert torch.equal(got.y[row], want.y[row])
    grad_x, _ = dense.rms_norm_backward(x.sign(), x, w, got.rstd)
    assert torch.isfinite(grad_x).all()


def test_blocks_that_are_not_finite_have_a_scale_that_is_none():
    from deepep_amd import dense

    rng = np.random.default_rng(15)
    x, w = _rows(rng, 4, 256, "bf16"), _weight(rng, 256, "bf16")
    want = dense.rms_norm(x, w, quantize="mxfp8")
    x[1, 7], x[2, 41] = float("nan"), float("-inf")
    got = dense.rms_norm(x, w, quantize="mxfp8")
    for row in (0, 3):
        assert torch.equal(got.codes[row].view(torch.uint8), want.codes[row].view(torch.uint8)) and torch.equal(got.scales[row], want.scales[row])
    assert (got.scales[1] == 255).all()
    # (an infinity's norm makes zeros of the other values and a NaN of it)
    assert got.scales[2, 1] == 255 and (got.scales[2] == 255).sum() == 1


def test_views_and_unaligned_rows():
    """Rows that start at an odd element are taken by way of a copy; rows that are not contiguous are refused."""
    from deepep_amd import dense

    rng = np.random.default_rng(6)
    x, w = _rows(rng, 3, 64, "bf16"), _weight(rng, 64, "bf16")
    shifted = torch.empty(3 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 64).copy_(x)
    assert shifted.data_ptr() % 16
    assert torch.equal(dense.rms_norm(shifted, w).y, dense.rms_norm(x, w).y)
    with pytest.raises(ValueError, match="contiguous"):
        dense.rms_norm(torch.cat([x, x], dim=1)[:, :64], w)


def test_parameters_that_require_gradients_are_taken():
    from deepep_amd import dense

    rng = np.random.default_rng(7)
    x, w = _rows(rng, 3, 64, "bf16"), _weight(rng, 64, "bf16")
    want = dense.rms_norm(x, w)
    got = dense.rms_norm(x, torch.nn.Parameter(w), eps=1e-6)
    assert torch.equal(got.y, want.y) and not got.y.requires_grad


def test_stream_in_place_through_the_c_abi():
    import ctypes

    from deepep_amd import _lib, dense, ops

    rng = np.random.default_rng(8)
    x, r, w = _rows(rng, 5, 2880, "bf16"), _rows(rng, 5, 2880, "bf16"), _weight(rng, 2880, "bf16")
    want = dense.rms_norm(x, w, r, eps=EPS)
    y = torch.empty_like(x)
    call = ops._Norm(x.data_ptr(), r.data_ptr(), w.data_ptr(), r.data_ptr(), y.data_ptr(), None, None, None, EPS, 1, 1, 0, 5, 2880)
    assert _lib.load().dpep_rms_norm(ctypes.byref(call), ops._stream(x.device)) == 0
    assert torch.equal(r, want.stream) and torch.equal(y, want.y)


def test_a_captured_step_replays():
    from deepep_amd import dense

    rng = np.random.default_rng(9)
    x, r, w = _rows(rng, 33, 1024, "bf16"), _rows(rng, 33, 1024, "bf16"), _weight(rng, 1024, "fp32")
    g = _rows(rng, 33, 1024, "bf16")

    def step():
        n = dense.rms_norm(x, w, r, quantize="fp8")
        return [n.y, n.stream, n.rstd, n.codes.view(torch.uint8), n.scales, *dense.rms_norm_backward(g, n.stream, w, n.rstd, g)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        x.copy_(_rows(rng, 33, 1024, "bf16"))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_another_stream():
    from deepep_amd import dense

    rng = np.random.default_rng(10)
    x, w = _rows(rng, 64, 4096, "bf16"), _weight(rng, 4096, "bf16")
    want = dense.rms_norm(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = dense.rms_norm(x, w)
    side.synchronize()
    assert torch.equal(got.y, want.y)
