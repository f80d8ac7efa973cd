"""What the norm, the gated block and the 8-bit products refuse before anything is launched; runs without a GPU."""

import ctypes

import pytest
import torch

from deepep_amd import _lib, dense, ops, w8


@pytest.fixture
def on_cpu(monkeypatch):
    """The checks of shapes and types with host tensors, as if they lived on the GPU; the library must not be reached."""
    def require(name, t, dtype, shape=None, device=None):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or not t.is_contiguous() or (shape is not None and tuple(t.shape) != tuple(shape)):
            raise ValueError(name)
        return t

    def load():
        raise AssertionError("reached the library")

    monkeypatch.setattr(ops, "_require", require)
    monkeypatch.setattr(ops._lib, "load", load)


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_host_tensors_are_refused():
    x, w = _bf16(2, 16), _bf16(16)
    for call in (lambda: dense.rms_norm(x, w), lambda: dense.rms_norm_backward(x, x, w, torch.zeros(2)), lambda: dense.gated_ffn(x, _bf16(32, 16), _bf16(16, 16)),
                 lambda: dense.gated_ffn_backward(x, x, _bf16(32, 16), _bf16(16, 16), torch.zeros(2, 32)), lambda: w8.quantize_tokens(x),
                 lambda: w8.matmul(x, w8.W8Weights(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)))):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("change", [
    dict(x=_bf16(2, 12)), dict(x=_bf16(2, 0)), dict(x=_bf16(16)), dict(x=_bf16(2, 16400)), dict(x=torch.zeros(2, 16, dtype=torch.int32)), dict(x=None),
    dict(x=_bf16(2, 32)[:, ::2]), dict(x=torch.zeros(2, 16, dtype=torch.float64)),
    dict(weight=_bf16(24)), dict(weight=torch.zeros(16, dtype=torch.float16)), dict(weight=None), dict(residual=_bf16(3, 16)), dict(residual=torch.zeros(2, 16)),
    dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=2), dict(eps="1"), dict(eps=True), dict(quantize="fp4"), dict(quantize="int8", x=_bf16(2, 24), weight=_bf16(24)),
    dict(quantize="mxfp8", x=_bf16(2, 16)), dict(quantize="fp8", x=_bf16(2, 8), weight=_bf16(8)), dict(output=False),
])
def test_norm_arguments(on_cpu, change):
    arguments = dict(x=_bf16(2, 16), weight=_bf16(16), residual=None, eps=1e-6, quantize=None, output=True) | change
    with pytest.raises(ValueError):
        ops.rms_norm(**arguments)


@pytest.mark.parametrize("change", [
    dict(grad_y=_bf16(3, 16)), dict(grad_y=torch.zeros(2, 16)), dict(stream=_bf16(2, 12)), dict(weight=_bf16(8)), dict(rstd=torch.zeros(3)), dict(rstd=_bf16(2)),
    dict(grad_stream=_bf16(2, 8)), dict(rstd=None),
])
def test_norm_backward_arguments(on_cpu, change):
    arguments = dict(grad_y=_bf16(2, 16), stream=_bf16(2, 16), weight=_bf16(16), rstd=torch.zeros(2), grad_stream=None) | change
    with pytest.raises(ValueError):
        ops.rms_norm_backward(**arguments)


@pytest.mark.parametrize("change", [
    dict(x=_bf16(2, 12)), dict(x=torch.zeros(2, 16)), dict(x=_bf16(2, 8)), dict(gate_up=_bf16(30, 16)), dict(gate_up=_bf16(48, 16)), dict(gate_up=torch.zeros(48, 16)),
    dict(down=_bf16(16, 20)), dict(down=_bf16(16, 0)), dict(down=_bf16(24)), dict(down=torch.zeros(16, 24, dtype=torch.float16)), dict(down=_bf16(24, 16).t()),
    dict(x=None), dict(gate_up=None),
])
@pytest.mark.parametrize("backward", [False, True])
def test_ffn_arguments(on_cpu, change, backward):
    arguments = dict(x=_bf16(2, 16), gate_up=_bf16(64, 16), down=_bf16(16, 32)) | change
    with pytest.raises((ValueError, AssertionError)) as raised:
        if backward:
            ops.gated_ffn_backward(_bf16(2, 16), kept=torch.zeros(2, 64), **arguments)
        else:
            ops.gated_ffn(**arguments)
    assert raised.type is ValueError or "reached" not in str(raised.value)


@pytest.mark.parametrize("change", [
    dict(x=_bf16(2, 8)), dict(x=_bf16(2, 32)), dict(x=(torch.zeros(2, 16, dtype=torch.int8),)), dict(x=(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(3))),
    dict(x=(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2))), dict(codes=torch.zeros(4, 24, dtype=torch.int8)), dict(codes=torch.zeros(0, 16, dtype=torch.int8)),
    dict(scales=torch.zeros(5)), dict(scales=_bf16(4)), dict(dtype=torch.int8), dict(dtype=torch.float64), dict(codes=torch.zeros(4, 65552, dtype=torch.int8)),
])
def test_w8_arguments(on_cpu, change):
    arguments = dict(x=_bf16(2, 16), codes=torch.zeros(4, 16, dtype=torch.int8), scales=torch.zeros(4)) | change
    with pytest.raises(ValueError):
        ops.w8_matmul(**arguments)


def _refused(status, text):
    assert status == -1
    assert text in _lib.load().dpep_last_error().decode()


def test_c_abi_refuses_before_it_launches():
    lib = _lib.load()
    at = 1 << 20  # (no call below reaches memory)
    norm = ops._Norm(at, None, 2 * at, None, 3 * at, 4 * at, None, None, 1e-6, 1, 1, 0, 4, 64)

    def norm_with(**change):
        call = ops._Norm.from_buffer_copy(norm)
        for name, value in change.items():
            setattr(call, name, value)
        return lib.dpep_rms_norm(ctypes.byref(call), None)

    assert norm_with(num_tokens=0) == 0
    _refused(norm_with(type=3), "type")
    _refused(norm_with(weight_type=2), "weight_type")
    _refused(norm_with(hidden=12), "H=12")
    _refused(norm_with(hidden=16392), "H=16392")
    _refused(norm_with(num_tokens=1 << 23), "T=")
    _refused(norm_with(num_tokens=-1), "T=")
    _refused(norm_with(quantize=4), "quantize")
    _refused(norm_with(quantize=1), "codes and scales")
    _refused(norm_with(quantize=2, hidden=48), "multiple of 32")
    _refused(norm_with(eps=-1.0), "eps")
    _refused(norm_with(eps=float("nan")), "eps")
    _refused(norm_with(residual=5 * at), "NULL")
    _refused(norm_with(stream_out=5 * at), "NULL")
    _refused(norm_with(x=at + 2), "misaligned")
    _refused(norm_with(y=at), "overlaps")
    _refused(norm_with(residual=5 * at, stream_out=5 * at + 64), "stream_out overlaps")
    _refused(norm_with(rstd=2 * at + 16), "overlaps")
    _refused(lib.dpep_rms_norm(None, None), "NULL")

    back = ops._NormGradients(at, 2 * at, 3 * at, 4 * at, None, 5 * at, 6 * at, 1, 1, 4, 64)

    def back_with(scratch=7 * at, **change):
        call = ops._NormGradients.from_buffer_copy(back)
        for name, value in change.items():
            setattr(call, name, value)
        return lib.dpep_rms_norm_backward(ctypes.byref(call), scratch, None)

    _refused(back_with(hidden=4), "H=4")
    _refused(back_with(scratch=None), "NULL")
    _refused(back_with(grad_weight=None), "NULL")
    _refused(back_with(grad_x=2 * at), "overlaps")
    _refused(back_with(grad_x=at + 32), "overlaps")
    _refused(back_with(grad_y=at + 8), "misaligned")

    ffn = ops._Ffn(at, 2 * at, 1, 64, 32)

    def ffn_with(x=3 * at, tokens=4, y=4 * at, kept=None, scratch=5 * at, **change):
        call = ops._Ffn.from_buffer_copy(ffn)
        for name, value in change.items():
            setattr(call, name, value)
        return lib.dpep_gated_ffn(ctypes.byref(call), x, tokens, y, kept, scratch, None)

    assert ffn_with(tokens=0) == 0
    _refused(ffn_with(type=0), "type")
    _refused(ffn_with(hidden=60), "H=60")
    _refused(ffn_with(inter=65544), "I=65544")
    _refused(ffn_with(tokens=1 << 21), "T=")
    _refused(ffn_with(gate_up=None), "NULL")
    _refused(ffn_with(y=3 * at + 16), "overlaps")
    _refused(ffn_with(kept=at), "overlaps")
    _refused(ffn_with(scratch=None), "NULL")
    _refused(lib.dpep_gated_ffn_backward(ctypes.byref(ffn), 3 * at, 4 * at, 5 * at, 4, 6 * at, 7 * at, 7 * at, 9 * at, None), "two outputs")
    _refused(lib.dpep_gated_ffn_backward(ctypes.byref(ffn), 3 * at, 4 * at, 5 * at, 4, 6 * at, at, 7 * at, 9 * at, None), "overlaps")
    _refused(lib.dpep_gated_ffn_backward(ctypes.byref(ffn), 3 * at, 4 * at, None, 4, 6 * at, 7 * at, 8 * at, 9 * at, None), "NULL")

    w = ops._W8(at, 2 * at, 8, 64)

    def w8_with(x=3 * at, x_scales=4 * at, rows=4, kind=1, y=5 * at, **change):
        call = ops._W8.from_buffer_copy(w)
        for name, value in change.items():
            setattr(call, name, value)
        return lib.dpep_w8_matmul(ctypes.byref(call), x, x_scales, rows, kind, y, 6 * at, None)

    assert w8_with(rows=0) == 0
    _refused(w8_with(kind=5), "type")
    _refused(w8_with(k=72), "K=72")
    _refused(w8_with(k=65552), "K=65552")
    _refused(w8_with(n=0), "N=0")
    _refused(w8_with(rows=-1), "T=-1")
    _refused(w8_with(x=3 * at + 4), "misaligned")
    _refused(w8_with(x=None), "NULL")
    _refused(w8_with(y=4 * at), "overlaps")
    _refused(lib.dpep_quantize_tokens(at, 1, 4, 24, 2 * at, 3 * at, None), "K=24")
    _refused(lib.dpep_quantize_tokens(at, 1, 4, 32, at + 16, 3 * at, None), "overlaps")
    _refused(lib.dpep_quantize_tokens(at, 4, 4, 32, 2 * at, 3 * at, None), "type")


def test_c_abi_refuses_what_overlaps():
    lib, at = _lib.load(), 1 << 20  # (no call below reaches memory)

    def norm(rstd=4 * at, codes=5 * at, scales=6 * at):
        return lib.dpep_rms_norm(ctypes.byref(ops._Norm(at, None, 2 * at, None, 3 * at, rstd, codes, scales, 1e-6, 1, 1, 3, 4, 64)), None)

    _refused(norm(scales=4 * at + 12), "another output")
    _refused(norm(codes=3 * at + 496), "another output")
    _refused(norm(rstd=6 * at), "another output")

    def backward(grad_x=5 * at, grad_weight=6 * at, scratch=7 * at):
        call = ops._NormGradients(at, 2 * at, 3 * at, 4 * at, None, grad_x, grad_weight, 1, 1, 4, 64)
        return lib.dpep_rms_norm_backward(ctypes.byref(call), scratch, None)

    _refused(backward(grad_weight=4 * at), "overlaps")
    _refused(backward(scratch=at), "overlaps")
    _refused(backward(scratch=5 * at + 256), "overlaps")
    _refused(backward(grad_weight=7 * at + 1008), "overlaps")

    ffn = ops._Ffn(at, 2 * at, 1, 64, 32)
    _refused(lib.dpep_gated_ffn(ctypes.byref(ffn), 3 * at, 4, 4 * at, None, 3 * at, None), "overlaps")
    _refused(lib.dpep_gated_ffn(ctypes.byref(ffn), 3 * at, 4, 4 * at, None, 4 * at + 16, None), "overlaps")
    _refused(lib.dpep_gated_ffn_backward(ctypes.byref(ffn), 3 * at, 4 * at, 5 * at, 4, 6 * at, 7 * at, 8 * at, 8 * at + 512, None), "overlaps")
    _refused(lib.dpep_gated_ffn_backward(ctypes.byref(ffn), 3 * at, 4 * at, 5 * at, 4, 6 * at, 7 * at, 8 * at, 5 * at, None), "overlaps")

    # (long rows: k in parts, whose sums are scratch)
    w = ops._W8(at, 3 * at, 300, 16384)
    far = 1 << 30
    assert lib.dpep_w8_matmul_scratch_bytes(300, 300, 16384) > 0
    _refused(lib.dpep_w8_matmul(ctypes.byref(w), far, 2 * far, 300, 1, 3 * far, far, None), "overlaps")
    _refused(lib.dpep_w8_matmul(ctypes.byref(w), far, 2 * far, 300, 1, 3 * far, 3 * far, None), "overlaps")
    _refused(lib.dpep_quantize_tokens(at, 1, 4, 32, 2 * at, 2 * at + 64, None), "other output")


def test_c_abi_refuses_scratch_that_is_not_aligned():
    """The parts' sums are stored and read 16 bytes at a time."""
    lib, far = _lib.load(), 1 << 30  # (no call below reaches memory)
    w = ops._W8(1 << 20, 3 << 20, 300, 16384)
    assert lib.dpep_w8_matmul_scratch_bytes(300, 300, 16384) > 0
    for off in (1, 4, 8):
        _refused(lib.dpep_w8_matmul(ctypes.byref(w), far, 2 * far, 300, 1, 3 * far, 4 * far + off, None), "scratch is NULL or misaligned")
    _refused(lib.dpep_w8_matmul(ctypes.byref(w), far, 2 * far, 300, 1, 3 * far, None, None), "scratch is NULL or misaligned")


def test_quantize_rounds_to_half_a_step():
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(5, 48, generator=gen)
    w[2] = 0
    got = w8.quantize(w)
    assert got.codes.dtype == torch.int8 and got.scales.dtype == torch.float32
    assert ((w8.dequantize(got) - w).abs() <= got.scales[:, None] * (0.5 + 1e-5)).all()
    assert (got.codes[2] == 0).all() and got.codes.abs().max() == 127
    with pytest.raises(ValueError):
        w8.quantize(w[0])
