"""Tensor-level entry points over the C-ABI (the counterpart of ``deep_ep._C`` in the reference,
csrc/bindings/module.cpp:17-95).

Like the reference's ``pointer()`` helper (csrc/ops/dispatch.cpp:36-49) every tensor is re-validated
here — device, dtype, contiguity, exact shape — before its address crosses the boundary.  Outputs
are allocated by the caller's framework (torch), never by the native side.  All calls enqueue on
torch's current stream and return without synchronising.
"""

from __future__ import annotations

import ctypes
import operator
from typing import Optional

import torch

from . import _lib


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device) -> ctypes.c_void_p:
    """torch's current stream on ``device`` as a raw hipStream_t."""
    if _raw_stream is not None and device.index is not None:
        return ctypes.c_void_p(_raw_stream(device.index))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class _on_device:
    """``torch.cuda.device(dev)`` that costs nothing when ``dev`` is already current (the usual case)."""

    __slots__ = ("guard",)

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def _require(name, t, dtype, shape=None, device=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on the GPU (got {t.device})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    return t


class Workspace:
    """Owner of the native HBM workspace."""

    def __init__(self, num_bytes: int, device: Optional[torch.device] = None):
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._lib = _lib.load()
        handle = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            _lib.check(self._lib.dpep_workspace_create(int(num_bytes), ctypes.byref(handle)), "workspace_create")
        self._handle = handle
        self.num_bytes = int(num_bytes)

    @property
    def handle(self):
        if self._handle is None:
            raise RuntimeError("workspace was destroyed")
        return self._handle

    @property
    def closed(self) -> bool:
        return self._handle is None

    def tune(self, key: str, value: int) -> None:
        """Test and diagnosis switches of the native workspace (``dpep_workspace_tune``)."""
        _lib.check(self._lib.dpep_workspace_tune(self.handle, key.encode(), int(value)), "workspace_tune")

    def destroy(self) -> None:
        if self._handle is not None:
            handle, self._handle = self._handle, None
            with torch.cuda.device(self.device):
                torch.cuda.synchronize(self.device)
                _lib.check(self._lib.dpep_workspace_destroy(handle), "workspace_destroy")


STORE_POLICIES = {"through": 0, "streaming": 1, "cached": 2}


def dispatch_store_policy(policy: Optional[str] = None) -> str:
    """Set (or, with no argument, read) how the dispatch kernels store their payload rows: ``"streaming"`` (default),
    ``"through"`` or ``"cached"``.  Process-wide.  Returns the policy that was in force before the call."""
    if policy is not None and policy not in STORE_POLICIES:
        raise ValueError(f"dispatch_store_policy: {policy!r} is not one of {sorted(STORE_POLICIES)}")
    code = _lib.load().dpep_dispatch_store_policy(3 if policy is None else STORE_POLICIES[policy])
    _lib.check(min(code, 0), "dispatch_store_policy")
    return {v: k for k, v in STORE_POLICIES.items()}[code]


def layout_workspace_bytes(num_tokens: int, num_topk: int, num_local: int) -> int:
    return int(_lib.load().dpep_layout_workspace_bytes(num_tokens, num_topk, num_local))


def layout(ws: Workspace, topk_idx: torch.Tensor, num_experts: int, expert_begin: int = 0, num_local: Optional[int] = None):
    """Routing layout on the device.  Returns device tensors; no host synchronisation.

    dict(counts[L], psum[L], offsets[L+1], route_to_row[T,K], row_to_route[T*K] (first R valid), num_rows[1]).
    """
    lib = _lib.load()
    _require("topk_idx", topk_idx, torch.int64, device=ws.device)
    if topk_idx.ndim != 2:
        raise ValueError("topk_idx must be [T, K]")
    tokens, topk = topk_idx.shape
    num_local = num_experts - expert_begin if num_local is None else num_local
    dev = topk_idx.device
    meta = torch.empty(3 * num_local + 2, dtype=torch.int32, device=dev)
    counts, psum = meta[:num_local], meta[num_local : 2 * num_local]
    offsets, num_rows = meta[2 * num_local : 3 * num_local + 1], meta[3 * num_local + 1 :]
    route_to_row = torch.empty((tokens, topk), dtype=torch.int32, device=dev)
    row_to_route = torch.empty((tokens * topk,), dtype=torch.int32, device=dev)
    with _on_device(dev):
        status = lib.dpep_layout(
            ws.handle, _ptr(topk_idx), tokens, topk, num_experts, expert_begin, num_local, _ptr(counts), _ptr(psum),
            _ptr(offsets), _ptr(route_to_row), _ptr(row_to_route), _ptr(num_rows), _stream(dev),
        )
    _lib.check(status, "layout")
    return dict(counts=counts, psum=psum, offsets=offsets, route_to_row=route_to_row, row_to_route=row_to_route,
                num_rows=num_rows, meta=meta)


def layout_wait(ws: Workspace, num_local: Optional[int] = None, timeout_s: float = 100.0):
    """The one host synchronisation of a fresh dispatch: waits for the most recent ``layout`` on ``ws`` and
    returns ``(counts, num_rows)`` as Python ints (``counts`` is None unless ``num_local`` is given).  The layout
    kernel writes these words into pinned host memory; nothing is copied and no stream is synchronised."""
    lib = _lib.load()
    rows = ctypes.c_int32()
    counts = None
    buf = None
    if num_local is not None:
        buf = (ctypes.c_int32 * num_local)()
    status = lib.dpep_layout_wait(ws.handle, buf, 0 if num_local is None else num_local, ctypes.byref(rows),
                                  int(timeout_s * 1e6))
    _lib.check(status, "layout_wait")
    if buf is not None:
        counts = list(buf)
    return counts, int(rows.value)


def dispatch_copy(x, scales, topk_weights, route_to_row, row_to_route, num_rows: Optional[int],
                  capacity_rows: Optional[int] = None):
    """out[row] = x[token(row)] (+ scale rows, + per-row weights).  x is BF16 [T,H] or FP8 [T,H].

    ``num_rows=None``: R is not known on the host yet (no ``layout_wait``): the outputs are allocated with T*K rows,
    (at least ``capacity_rows``, if given), of which the first R are written; the caller narrows them."""
    lib = _lib.load()
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bfloat16, torch.float8_e4m3fn, torch.float16):
        raise ValueError("x must be a BF16, FP16 or FP8 E4M3FN tensor")
    _require("x", x, x.dtype)
    if x.ndim != 2:
        raise ValueError("x must be [T, H]")
    dev = x.device
    tokens, hidden = x.shape
    _require("route_to_row", route_to_row, torch.int32, device=dev)
    topk = route_to_row.shape[1]
    _require("route_to_row", route_to_row, torch.int32, (tokens, topk), dev)
    _require("row_to_route", row_to_route, torch.int32, device=dev)
    row_bytes = hidden * x.element_size()
    if row_bytes % 16:
        raise ValueError("hidden row size must be a multiple of 16 bytes")
    num_rows, known_rows = (max(tokens * topk, capacity_rows or 0), -1) if num_rows is None else (num_rows, num_rows)
    scale_cols = 0
    out_scales = None
    if scales is not None:
        # FP32 scales, or int32 words holding four packed E8M0 bytes (the low-latency scale format,
        # docs/elastic.md:97): either way 4-byte words that are moved bit for bit
        if not isinstance(scales, torch.Tensor) or scales.dtype not in (torch.float32, torch.int32):
            raise ValueError("scales must be FP32 or packed int32")
        _require("scales", scales, scales.dtype, device=dev)
        if scales.ndim != 2 or scales.shape[0] != tokens:
            raise ValueError("scales must be [T, C]")
        scale_cols = scales.shape[1]
        out_scales = torch.empty((num_rows, scale_cols), dtype=scales.dtype, device=dev)
    out_weights = None
    if topk_weights is not None:
        _require("topk_weights", topk_weights, torch.float32, (tokens, topk), dev)
        out_weights = torch.empty((num_rows,), dtype=torch.float32, device=dev)
    out = torch.empty((num_rows, hidden), dtype=x.dtype, device=dev)
    with _on_device(dev):
        status = lib.dpep_dispatch_copy(
            _ptr(x), _ptr(scales), _ptr(topk_weights), _ptr(route_to_row), _ptr(row_to_route), tokens, topk, known_rows,
            row_bytes, scale_cols, _ptr(out), _ptr(out_scales), _ptr(out_weights), _stream(dev),
        )
    _lib.check(status, "dispatch_copy")
    return out, out_scales, out_weights


SMALL_BATCH_ROUTES = 2048  # T*K up to which layout and dispatch share one launch (dpep_layout_dispatch_small)


def layout_dispatch_small(ws: Workspace, topk_idx, x, scales, topk_weights, num_experts: int, expert_begin: int = 0,
                          num_local: Optional[int] = None, quantize: bool = False, capacity_rows: Optional[int] = None):
    """Routing layout and payload dispatch of a small batch in one launch (``1 <= T*K <= SMALL_BATCH_ROUTES``).

    Returns ``(layout, out, out_scales, out_weights)``: ``layout`` as from ``layout()`` (``layout_wait`` works on it),
    the payload outputs as from ``dispatch_copy`` / ``dispatch_quant_fp8`` with ``num_rows=None``: allocated with T*K rows
    (at least ``capacity_rows``), of which the first R are written."""
    lib = _lib.load()
    _require("topk_idx", topk_idx, torch.int64, device=ws.device)
    if topk_idx.ndim != 2:
        raise ValueError("topk_idx must be [T, K]")
    tokens, topk = topk_idx.shape
    if not 1 <= tokens * topk <= SMALL_BATCH_ROUTES:
        raise ValueError(f"layout_dispatch_small takes 1..{SMALL_BATCH_ROUTES} routes")
    dev = topk_idx.device
    allowed = (torch.bfloat16,) if quantize else (torch.bfloat16, torch.float8_e4m3fn, torch.float16)
    if not isinstance(x, torch.Tensor) or x.dtype not in allowed:
        raise ValueError("x must be BF16 (quantize) or a BF16, FP16 or FP8 E4M3FN tensor")
    _require("x", x, x.dtype, device=dev)
    if x.ndim != 2 or x.shape[0] != tokens:
        raise ValueError("x must be [T, H]")
    hidden = x.shape[1]
    row_bytes = hidden * x.element_size()
    if quantize and hidden % 128:
        raise ValueError("hidden must be a multiple of 128 for FP8 dispatch")
    if row_bytes % 16:
        raise ValueError("hidden row size must be a multiple of 16 bytes")
    num_local = num_experts - expert_begin if num_local is None else num_local
    rows = max(tokens * topk, capacity_rows or 0)
    meta = torch.empty(3 * num_local + 2, dtype=torch.int32, device=dev)
    counts, psum = meta[:num_local], meta[num_local : 2 * num_local]
    offsets, num_rows = meta[2 * num_local : 3 * num_local + 1], meta[3 * num_local + 1 :]
    route_to_row = torch.empty((tokens, topk), dtype=torch.int32, device=dev)
    row_to_route = torch.empty((tokens * topk,), dtype=torch.int32, device=dev)
    scale_cols = 0
    out_scales = None
    if quantize:
        if scales is not None:
            raise ValueError("the fused quantiser takes no input scales")
        out = torch.empty((rows, hidden), dtype=torch.float8_e4m3fn, device=dev)
        out_scales = torch.empty((rows, hidden // 128), dtype=torch.float32, device=dev)
    else:
        out = torch.empty((rows, hidden), dtype=x.dtype, device=dev)
        if scales is not None:
            if not isinstance(scales, torch.Tensor) or scales.dtype not in (torch.float32, torch.int32):
                raise ValueError("scales must be FP32 or packed int32")
            _require("scales", scales, scales.dtype, device=dev)
            if scales.ndim != 2 or scales.shape[0] != tokens:
                raise ValueError("scales must be [T, C]")
            scale_cols = scales.shape[1]
            out_scales = torch.empty((rows, scale_cols), dtype=scales.dtype, device=dev)
    out_weights = None
    if topk_weights is not None:
        _require("topk_weights", topk_weights, torch.float32, (tokens, topk), dev)
        out_weights = torch.empty((rows,), dtype=torch.float32, device=dev)
    with _on_device(dev):
        status = lib.dpep_layout_dispatch_small(
            ws.handle, _ptr(topk_idx), _ptr(x), _ptr(scales), _ptr(topk_weights), tokens, topk, num_experts, expert_begin,
            num_local, row_bytes, scale_cols, int(bool(quantize)), _ptr(counts), _ptr(psum), _ptr(offsets), _ptr(route_to_row),
            _ptr(row_to_route), _ptr(num_rows), _ptr(out), _ptr(out_scales), _ptr(out_weights), _stream(dev),
        )
    _lib.check(status, "layout_dispatch_small")
    layout_out = dict(counts=counts, psum=psum, offsets=offsets, route_to_row=route_to_row, row_to_route=row_to_route,
                      num_rows=num_rows, meta=meta)
    return layout_out, out, out_scales, out_weights


def dispatch_quant_fp8(x, topk_weights, route_to_row, row_to_route, num_rows: Optional[int]):
    """Fused per-128 FP8 quantisation + expand-permute of BF16 x [T,H]; ``num_rows=None`` as in ``dispatch_copy``."""
    lib = _lib.load()
    _require("x", x, torch.bfloat16)
    if x.ndim != 2:
        raise ValueError("x must be [T, H]")
    dev = x.device
    tokens, hidden = x.shape
    if hidden % 128:
        raise ValueError("hidden must be a multiple of 128 for FP8 dispatch")
    _require("route_to_row", route_to_row, torch.int32, device=dev)
    topk = route_to_row.shape[1]
    _require("route_to_row", route_to_row, torch.int32, (tokens, topk), dev)
    _require("row_to_route", row_to_route, torch.int32, device=dev)
    num_rows, known_rows = (tokens * topk, -1) if num_rows is None else (num_rows, num_rows)
    out_weights = None
    if topk_weights is not None:
        _require("topk_weights", topk_weights, torch.float32, (tokens, topk), dev)
        out_weights = torch.empty((num_rows,), dtype=torch.float32, device=dev)
    out = torch.empty((num_rows, hidden), dtype=torch.float8_e4m3fn, device=dev)
    out_scales = torch.empty((num_rows, hidden // 128), dtype=torch.float32, device=dev)
    with _on_device(dev):
        status = lib.dpep_dispatch_quant_fp8(
            _ptr(x), _ptr(topk_weights), _ptr(route_to_row), _ptr(row_to_route), tokens, topk, known_rows, hidden,
            _ptr(out), _ptr(out_scales), _ptr(out_weights), _stream(dev),
        )
    _lib.check(status, "dispatch_quant_fp8")
    return out, out_scales, out_weights


def cast_to_fp8(x):
    """per_token_cast_to_fp8 on the device: BF16 [T,H] -> (FP8 [T,H], FP32 [T,ceil(H/128)]); a short last block is
    quantised as if padded with zeros, as the reference does."""
    lib = _lib.load()
    _require("x", x, torch.bfloat16)
    if x.ndim != 2 or x.shape[1] % 16 or x.shape[1] == 0:
        raise ValueError("x must be [T, H] with H a positive multiple of 16")
    tokens, hidden = x.shape
    out = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((tokens, (hidden + 127) // 128), dtype=torch.float32, device=x.device)
    with _on_device(x.device):
        status = lib.dpep_cast_to_fp8(_ptr(x), tokens, hidden, _ptr(out), _ptr(scales), _stream(x.device))
    _lib.check(status, "cast_to_fp8")
    return out, scales


def cast_back(codes, scales):
    """per_token_cast_back on the device: (FP8 e4m3fn [T,H], scales) -> BF16 [T,H], bf16(fp32(code) * scale) per block of
    128 columns.  scales: FP32 [T, ceil(H/128)], or int32 [T, ceil(H/128)/4] holding four e8m0 exponent bytes each."""
    lib = _lib.load()
    _require("codes", codes, torch.float8_e4m3fn)
    if codes.ndim != 2 or codes.shape[1] % 16 or codes.shape[1] == 0:
        raise ValueError("codes must be [T, H] with H a positive multiple of 16")
    tokens, hidden = codes.shape
    blocks = (hidden + 127) // 128
    if scales.dtype == torch.int32:
        if blocks % 4:
            raise ValueError("int32 scales hold four blocks each: ceil(H/128) must be a multiple of 4")
        _require("scales", scales, torch.int32, (tokens, blocks // 4), codes.device)
    else:
        _require("scales", scales, torch.float32, (tokens, blocks), codes.device)
    out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=codes.device)
    with _on_device(codes.device):
        status = lib.dpep_cast_back(_ptr(codes), _ptr(scales), int(scales.dtype == torch.int32), tokens, hidden, _ptr(out),
                                    _stream(codes.device))
    _lib.check(status, "cast_back")
    return out


def combine(y, route_to_row, row_weights=None, return_values=None, out=None, served_only=False):
    """out[t] = round( sum_s fp32(y[row(t,s)]) (* row_weights[row]) ) in y's dtype (BF16 or FP16); optional
    weight-return channel.  ``served_only`` (BF16, needs ``out``): tokens without any row keep what ``out`` held instead
    of being zero-filled (one rank's share of an EP job produces nothing for the tokens it does not serve)."""
    lib = _lib.load()
    if not isinstance(y, torch.Tensor) or y.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("y must be a BF16 or FP16 tensor")
    _require("y", y, y.dtype)
    if y.ndim != 2:
        raise ValueError("y must be [R, H]")
    dev = y.device
    rows, hidden = y.shape
    if hidden % 8:
        raise ValueError("hidden must be a multiple of 8")
    _require("route_to_row", route_to_row, torch.int32, device=dev)
    if route_to_row.ndim != 2:
        raise ValueError("route_to_row must be [T, K]")
    tokens, topk = route_to_row.shape
    if row_weights is not None:
        _require("row_weights", row_weights, torch.float32, (rows,), dev)
    returned = None
    if return_values is not None:
        _require("return_values", return_values, torch.float32, (rows,), dev)
        returned = torch.empty((tokens, topk), dtype=torch.float32, device=dev)
    if out is None:
        if served_only:
            raise ValueError("served_only needs the caller's out (rows of unserved tokens are left as they are)")
        out = torch.empty((tokens, hidden), dtype=y.dtype, device=dev)
    else:
        _require("out", out, y.dtype, (tokens, hidden), dev)
    entry = lib.dpep_combine if y.dtype == torch.bfloat16 else lib.dpep_combine_fp16
    if served_only:
        if y.dtype != torch.bfloat16:
            raise ValueError("served_only is available for BF16 rows")
        entry = lib.dpep_combine_served
    with _on_device(dev):
        status = entry(
            _ptr(y), _ptr(row_weights), _ptr(route_to_row), tokens, topk, rows, hidden, _ptr(out),
            _ptr(return_values), _ptr(returned), _stream(dev),
        )
    _lib.check(status, "combine")
    return out, returned


# ---------------------------------------------------------------------------------------------
# MegaMoE (W4A8) entry points
# ---------------------------------------------------------------------------------------------
def mx_quant(x):
    """MXFP8 activation quantiser: BF16 [B,H] -> (e4m3 codes [B,H] as float8_e4m3fn, e8m0 bytes [B,H/32] uint8)."""
    lib = _lib.load()
    _require("x", x, torch.bfloat16)
    if x.ndim != 2 or x.shape[1] % 32:
        raise ValueError("x must be [B, H] with H a multiple of 32")
    rows, hidden = x.shape
    codes = torch.empty((rows, hidden), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((rows, hidden // 32), dtype=torch.uint8, device=x.device)
    with _on_device(x.device):
        status = lib.dpep_mx_quant(_ptr(x), rows, hidden, _ptr(codes), _ptr(scales), _stream(x.device))
    _lib.check(status, "mx_quant")
    return codes, scales


def megamoe_workspace_bytes(num_tokens, num_topk, hidden, intermediate, num_local, num_shared: int = 0) -> int:
    return int(_lib.load().dpep_megamoe_workspace_bytes(num_tokens, num_topk, hidden, intermediate, num_local, num_shared))


def megamoe_padded_dim(dim: int) -> int:
    """What the grouped GEMM works on for a logical hidden / intermediate size (whole 256-column tiles, at least 512)."""
    return int(_lib.load().dpep_megamoe_padded_dim(int(dim)))


def megamoe_prepared_shape(n: int, k: int, gate_up: bool):
    """(padded N, padded K, scale bytes per column) of the prepared form of a raw [L,N,K/2] weight tensor."""
    import ctypes

    out = [ctypes.c_int(0) for _ in range(3)]
    status = _lib.load().dpep_megamoe_prepared_shape(int(n), int(k), int(bool(gate_up)), *(ctypes.byref(v) for v in out))
    _lib.check(status, "megamoe_prepared_shape")
    return tuple(v.value for v in out)


def megamoe_prepare_weights(w_packed, w_scales, gate_up: bool):
    """Raw packed FP4 uint8 [L,N,K/2] + e8m0 uint8 [L,N,K/32] -> the kernel's streaming order, padded to the sizes the
    GEMM works on (``megamoe_prepared_shape``: zero codes and unit scales behind N and K).

    Returns (packed [L,Np,Kp/2], scales [L,Np,scale_cols])."""
    lib = _lib.load()
    _require("w_packed", w_packed, torch.uint8)
    if w_packed.ndim != 3:
        raise ValueError("w_packed must be [L, N, K/2]")
    experts, n, half_k = w_packed.shape
    k = half_k * 2
    _require("w_scales", w_scales.reshape(experts, n, -1), torch.uint8, (experts, n, k // 32), w_packed.device)
    np_, kp, scale_cols = megamoe_prepared_shape(n, k, gate_up)
    out_w = torch.empty((experts, np_, kp // 2), dtype=torch.uint8, device=w_packed.device)
    out_s = torch.empty((experts, np_, scale_cols), dtype=torch.uint8, device=w_packed.device)
    with _on_device(w_packed.device):
        status = lib.dpep_megamoe_prepare_weights(
            _ptr(w_packed), _ptr(w_scales), experts, n, k, int(bool(gate_up)), _ptr(out_w), _ptr(out_s),
            _stream(w_packed.device),
        )
    _lib.check(status, "megamoe_prepare_weights")
    return out_w, out_s


def megamoe_gemm_choice(num_tokens: int, hidden: int, intermediate: int, num_topk: int, num_experts: int, num_local: int,
                        num_shared: int = 0, ws: Optional[Workspace] = None):
    """``((tile rows, waves per workgroup) of the first GEMM, the same of the second)`` that a forward of these sizes takes;
    32 rows: the kernel for few rows per expert.  Host arithmetic only."""
    chosen = []
    for second in (0, 1):
        rows, waves = ctypes.c_int32(), ctypes.c_int32()
        status = _lib.load().dpep_megamoe_gemm_choice(None if ws is None else ws.handle, num_tokens, hidden, intermediate, num_topk, num_experts,
                                                      num_local, num_shared, second, ctypes.byref(rows), ctypes.byref(waves))
        _lib.check(status, "megamoe_gemm_choice")
        chosen.append((rows.value, waves.value))
    return tuple(chosen)


GEMM_KERNELS = ("two_by_two", "column_waves", "paired", "paired_streamed", "few_rows", "one_wave")


def megamoe_gemm_kernels(num_tokens: int, hidden: int, intermediate: int, num_topk: int, num_experts: int, num_local: int,
                         num_shared: int = 0, ws: Optional[Workspace] = None):
    """The kernels (names of ``GEMM_KERNELS``) that a forward of these sizes takes for its first and its second GEMM.  Host arithmetic only."""
    kernels = []
    for second in (0, 1):
        kernel = ctypes.c_int32()
        status = _lib.load().dpep_megamoe_gemm_kernel(None if ws is None else ws.handle, num_tokens, hidden, intermediate, num_topk, num_experts,
                                                      num_local, num_shared, second, ctypes.byref(kernel))
        _lib.check(status, "megamoe_gemm_kernel")
        kernels.append(GEMM_KERNELS[kernel.value])
    return tuple(kernels)


def megamoe_fill_report(ws, num_tokens, num_topk, hidden, intermediate, num_local, num_shared: int = 0):
    """(filler waves, tokens they looked at) of the most recent forward on ``ws``; waits for the current stream."""
    fillers, filled = ctypes.c_int32(0), ctypes.c_int64(0)
    device = ws.device
    status = _lib.load().dpep_megamoe_fill_report(ws.handle, num_tokens, num_topk, hidden, intermediate, num_local, num_shared,
                                                  ctypes.byref(fillers), ctypes.byref(filled), _stream(device))
    _lib.check(status, "megamoe_fill_report")
    return fillers.value, filled.value


def megamoe_forward(ws, x_codes, x_scales, topk_idx, topk_weights, w1, s1, w2, s2, num_experts, expert_begin,
                    num_local, y, expert_token_nums, shared=None, intermediate=None):
    """Fused W4A8 forward of one rank's local experts; writes y [B,H] BF16 and expert_token_nums [L] int32.

    ``intermediate`` = the experts' logical intermediate size; by default what the prepared ``w1`` holds (right unless
    the weights were padded).  ``shared`` = (w1, s1, w2, s2) prepared weights of S shared experts, which every token
    passes through."""
    lib = _lib.load()
    dev = ws.device
    _require("x_codes", x_codes, torch.float8_e4m3fn, device=dev)
    tokens, hidden = x_codes.shape
    _require("x_scales", x_scales, torch.uint8, (tokens, hidden // 32), dev)
    _require("topk_idx", topk_idx, torch.int32, device=dev)
    topk = topk_idx.shape[1]
    _require("topk_idx", topk_idx, torch.int32, (tokens, topk), dev)
    _require("topk_weights", topk_weights, torch.float32, (tokens, topk), dev)
    _require("w1", w1, torch.uint8, device=dev)
    if w1.ndim != 3 or w1.shape[0] != num_local or w1.shape[1] % 2:
        raise ValueError("w1 must be prepared [L, 2I, H/2]")
    if intermediate is None:
        intermediate = w1.shape[1] // 2
    if hidden % 64 or intermediate % 128 or hidden < 64 or intermediate < 128:
        raise ValueError("hidden must be a positive multiple of 64, intermediate of 128")
    n1, k1, cols1 = megamoe_prepared_shape(2 * intermediate, hidden, True)
    n2, k2, cols2 = megamoe_prepared_shape(hidden, intermediate, False)
    _require("w1", w1, torch.uint8, (num_local, n1, k1 // 2), dev)
    _require("s1", s1, torch.uint8, (num_local, n1, cols1), dev)
    _require("w2", w2, torch.uint8, (num_local, n2, k2 // 2), dev)
    _require("s2", s2, torch.uint8, (num_local, n2, cols2), dev)
    _require("y", y, torch.bfloat16, (tokens, hidden), dev)
    _require("expert_token_nums", expert_token_nums, torch.int32, (num_local,), dev)
    num_shared = 0
    sw1 = ss1 = sw2 = ss2 = None
    if shared is not None:
        sw1, ss1, sw2, ss2 = shared
        _require("shared w1", sw1, torch.uint8, device=dev)
        num_shared = sw1.shape[0]
        _require("shared w1", sw1, torch.uint8, (num_shared, n1, k1 // 2), dev)
        _require("shared s1", ss1, torch.uint8, (num_shared, n1, cols1), dev)
        _require("shared w2", sw2, torch.uint8, (num_shared, n2, k2 // 2), dev)
        _require("shared s2", ss2, torch.uint8, (num_shared, n2, cols2), dev)
    with _on_device(dev):
        status = lib.dpep_megamoe_forward(
            ws.handle, _ptr(x_codes), _ptr(x_scales), _ptr(topk_idx), _ptr(topk_weights), _ptr(w1), _ptr(s1), _ptr(w2),
            _ptr(s2), _ptr(sw1), _ptr(ss1), _ptr(sw2), _ptr(ss2), num_shared, tokens, hidden, intermediate, topk,
            num_experts, expert_begin, num_local, _ptr(y), _ptr(expert_token_nums), _stream(dev),
        )
    _lib.check(status, "megamoe_forward")
    return y, expert_token_nums


# ---------------------------------------------------------------------------------------------
# Router, balance loss and 4-bit products
# ---------------------------------------------------------------------------------------------
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # DPEP_TYPE_*
SCORES = ("softmax", "sigmoid")  # DPEP_SCORE_*
_MAX_ROUTER_TOKENS, _MAX_SEQUENCES, _MAX_ROUTES = 1 << 30, (1 << 22) - 1, (1 << 31) - 1  # DPEP_MAX_*; routes of a balance loss
_W4_MAX_N, _W4_MAX_K, _W4_MAX_ROWS, _W4_MAX_ROUTES, _MAX_LOCAL_EXPERTS, _MAX_TOPK = 1 << 30, 16384, 65535, 2048, 1024, 32  # DPEP_*


class RouterSpec(ctypes.Structure):
    """``dpep_router`` of include/deepep_amd.h."""

    _fields_ = [("num_experts", ctypes.c_int32), ("num_topk", ctypes.c_int32), ("num_groups", ctypes.c_int32),
                ("num_topk_groups", ctypes.c_int32), ("score", ctypes.c_int32), ("normalize", ctypes.c_int32),
                ("scale", ctypes.c_float), ("logits_type", ctypes.c_int32), ("index_bytes", ctypes.c_int32)]


class _RouterGradients(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("logits", "topk_idx", "topk_weights", "grad_weights", "sequence_offsets", "counts",
                                                     "tokens", "grad_losses", "grad_logits")] + [("num_sequences", ctypes.c_int32)]


class _W4(ctypes.Structure):
    _fields_ = [("packed", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("zeros", ctypes.c_void_p),
                ("n", ctypes.c_int32), ("k", ctypes.c_int32), ("group", ctypes.c_int32)]


def _at_most(limit, **sizes):
    """Sizes are compared as Python holds them: the C struct or call that they go into would keep 32 bits of them, and the outputs and
    scratch of a call that is refused need not be allocated."""
    for name, size in sizes.items():
        if size > limit:
            raise ValueError(f"{name}={size} is more than {limit}")


def _require_logits(spec: RouterSpec, logits):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _TYPES:
        raise ValueError("logits must be an FP32, BF16 or FP16 tensor")
    _require("logits", logits, logits.dtype)
    if logits.ndim != 2 or logits.shape[1] != spec.num_experts:
        raise ValueError(f"logits must be [T, {spec.num_experts}] (got {tuple(logits.shape)})")
    _at_most(_MAX_ROUTER_TOKENS, tokens=logits.shape[0])
    spec.logits_type = _TYPES[logits.dtype]
    return logits.shape[0], logits.device


def _require_routes(spec: RouterSpec, topk_idx, tokens, device):
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("topk_idx must be an int64 or int32 tensor")
    _require("topk_idx", topk_idx, topk_idx.dtype, (tokens, spec.num_topk), device)
    spec.index_bytes = topk_idx.element_size()


def _require_sequences(spec: RouterSpec, tokens, sequence_offsets, device):
    _at_most(_MAX_ROUTES, routes=tokens * spec.num_topk)
    if sequence_offsets is None:
        return 1
    _require("sequence_offsets", sequence_offsets, torch.int32, device=device)
    if sequence_offsets.ndim != 1 or sequence_offsets.shape[0] < 2:
        raise ValueError("sequence_offsets must be [B + 1] with B >= 1")
    _at_most(_MAX_SEQUENCES, sequences=sequence_offsets.shape[0] - 1)
    return sequence_offsets.shape[0] - 1


def route(spec: RouterSpec, logits, bias=None, token_mask=None, index_dtype=torch.int64):
    """``(topk_idx [T,K], topk_weights FP32 [T,K])`` of logits [T,E]; ``bias`` FP32 [E], ``token_mask`` bool [T] (False: padding)."""
    tokens, dev = _require_logits(spec, logits)
    if index_dtype not in (torch.int64, torch.int32):
        raise ValueError("index_dtype must be torch.int64 or torch.int32")
    if bias is not None:
        _require("bias", bias, torch.float32, (spec.num_experts,), dev)
    if token_mask is not None:
        _require("token_mask", token_mask, torch.bool, (tokens,), dev)
    spec.index_bytes = 8 if index_dtype == torch.int64 else 4
    topk_idx = torch.empty((tokens, spec.num_topk), dtype=index_dtype, device=dev)
    topk_weights = torch.empty((tokens, spec.num_topk), dtype=torch.float32, device=dev)
    with _on_device(dev):
        status = _lib.load().dpep_route(ctypes.byref(spec), _ptr(logits), _ptr(bias), _ptr(token_mask), tokens, _ptr(topk_idx),
                                        _ptr(topk_weights), _stream(dev))
    _lib.check(status, "route")
    return topk_idx, topk_weights


def balance_loss(spec: RouterSpec, logits, topk_idx, sequence_offsets=None):
    """``(losses FP32 [B], counts int32 [B,E], tokens int32 [B])`` of the sequences that ``sequence_offsets`` int32 [B+1] cuts the
    batch into (None: one)."""
    tokens, dev = _require_logits(spec, logits)
    _require_routes(spec, topk_idx, tokens, dev)
    sequences = _require_sequences(spec, tokens, sequence_offsets, dev)
    lib = _lib.load()
    losses = torch.empty((sequences,), dtype=torch.float32, device=dev)
    counts = torch.empty((sequences, spec.num_experts), dtype=torch.int32, device=dev)
    members = torch.empty((sequences,), dtype=torch.int32, device=dev)
    scratch = torch.empty((lib.dpep_balance_scratch_bytes(spec.num_experts, tokens, sequences),), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        status = lib.dpep_balance_loss(ctypes.byref(spec), _ptr(logits), _ptr(topk_idx), tokens, _ptr(sequence_offsets), sequences,
                                       _ptr(losses), _ptr(counts), _ptr(members), _ptr(scratch), _stream(dev))
    _lib.check(status, "balance_loss")
    return losses, counts, members


def route_balance(spec: RouterSpec, logits, bias=None, token_mask=None, sequence_offsets=None, index_dtype=torch.int64):
    """``route`` and the ``balance_loss`` of its routes in one pass: ``(topk_idx, topk_weights, losses, counts, tokens)``."""
    tokens, dev = _require_logits(spec, logits)
    if index_dtype not in (torch.int64, torch.int32):
        raise ValueError("index_dtype must be torch.int64 or torch.int32")
    if bias is not None:
        _require("bias", bias, torch.float32, (spec.num_experts,), dev)
    if token_mask is not None:
        _require("token_mask", token_mask, torch.bool, (tokens,), dev)
    sequences = _require_sequences(spec, tokens, sequence_offsets, dev)
    spec.index_bytes = 8 if index_dtype == torch.int64 else 4
    lib = _lib.load()
    topk_idx = torch.empty((tokens, spec.num_topk), dtype=index_dtype, device=dev)
    topk_weights = torch.empty((tokens, spec.num_topk), dtype=torch.float32, device=dev)
    losses = torch.empty((sequences,), dtype=torch.float32, device=dev)
    counts = torch.empty((sequences, spec.num_experts), dtype=torch.int32, device=dev)
    members = torch.empty((sequences,), dtype=torch.int32, device=dev)
    scratch = torch.empty((lib.dpep_balance_scratch_bytes(spec.num_experts, tokens, sequences),), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        status = lib.dpep_route_balance(ctypes.byref(spec), _ptr(logits), _ptr(bias), _ptr(token_mask), tokens, _ptr(sequence_offsets), sequences,
                                        _ptr(topk_idx), _ptr(topk_weights), _ptr(losses), _ptr(counts), _ptr(members), _ptr(scratch), _stream(dev))
    _lib.check(status, "route_balance")
    return topk_idx, topk_weights, losses, counts, members


def router_backward(spec: RouterSpec, logits, topk_idx, topk_weights=None, grad_weights=None, sequence_offsets=None, counts=None,
                    tokens=None, grad_losses=None):
    """Gradient of ``logits`` in their type, from ``grad_weights`` FP32 [T,K], from ``grad_losses`` FP32 [B] with what
    ``balance_loss`` was given and returned, or from both."""
    num_tokens, dev = _require_logits(spec, logits)
    _require_routes(spec, topk_idx, num_tokens, dev)
    if grad_weights is None and grad_losses is None:
        raise ValueError("router_backward needs grad_weights, grad_losses or both")
    sequences = 1
    if grad_weights is not None:
        _require("grad_weights", grad_weights, torch.float32, (num_tokens, spec.num_topk), dev)
        if spec.normalize:
            _require("topk_weights", topk_weights, torch.float32, (num_tokens, spec.num_topk), dev)
    if grad_losses is not None:
        sequences = _require_sequences(spec, num_tokens, sequence_offsets, dev)
        _require("grad_losses", grad_losses, torch.float32, (sequences,), dev)
        _require("counts", counts, torch.int32, (sequences, spec.num_experts), dev)
        _require("tokens", tokens, torch.int32, (sequences,), dev)
    grad_logits = torch.empty_like(logits)
    address = [None if t is None else t.data_ptr() for t in (logits, topk_idx, topk_weights, grad_weights, sequence_offsets, counts, tokens,
                                                             grad_losses, grad_logits)]
    call = _RouterGradients(*address, sequences)
    with _on_device(dev):
        status = _lib.load().dpep_router_backward(ctypes.byref(spec), ctypes.byref(call), num_tokens, _stream(dev))
    _lib.check(status, "router_backward")
    return grad_logits


def _w4(name, packed, scales, zeros, dtype, device, ndim):
    """The C struct of a matrix ([N,K/2]) or of experts' matrices ([L,N,K/2])."""
    _require(f"{name} packed", packed, torch.uint8, device=device)
    if packed.ndim != ndim or packed.shape[-1] == 0 or packed.shape[-2] == 0:
        raise ValueError(f"{name} packed must be [{'L, ' if ndim == 3 else ''}N, K/2]")
    _require(f"{name} scales", scales, dtype, device=device)
    k, groups = 2 * packed.shape[-1], scales.shape[-1] if scales.ndim == ndim else 0
    if scales.ndim != ndim or scales.shape[:-1] != packed.shape[:-1] or groups == 0 or k % groups:
        raise ValueError(f"{name} scales must be {tuple(packed.shape[:-1])} + (K / group,) (got {tuple(scales.shape)})")
    if zeros is not None:
        _require(f"{name} zeros", zeros, torch.uint8, tuple(scales.shape), device)
    _at_most(_W4_MAX_N, N=packed.shape[-2])
    _at_most(_W4_MAX_K, K=k)
    return _W4(packed.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), packed.shape[-2], k, k // groups)


def _aligned(x):
    return x if x.data_ptr() % 16 == 0 else x.clone()


def w4_matvec(x, packed, scales, zeros=None, out=None):
    """x [M,K] (BF16 or FP16) times a matrix of 4-bit values: packed uint8 [N,K/2], scales [N,K/group] in x's type, zeros uint8
    [N,K/group] (None: 8).  Returns [M,N] in x's type."""
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x must be a BF16 or FP16 tensor")
    _require("x", x, x.dtype)
    dev = x.device
    weights = _w4("w4_matvec", packed, scales, zeros, x.dtype, dev, 2)
    if x.ndim != 2 or x.shape[1] != weights.k:
        raise ValueError(f"x must be [M, {weights.k}] (got {tuple(x.shape)})")
    rows = x.shape[0]
    _at_most(_W4_MAX_ROWS, rows=rows)
    if out is None:
        out = torch.empty((rows, weights.n), dtype=x.dtype, device=dev)
    else:
        _require("out", out, x.dtype, (rows, weights.n), dev)
    x = _aligned(x)
    with _on_device(dev):
        status = _lib.load().dpep_w4_matvec(ctypes.byref(weights), _TYPES[x.dtype], _ptr(x), rows, _ptr(out), _stream(dev))
    _lib.check(status, "w4_matvec")
    return out


def w4_experts(x, topk_idx, topk_weights, gate_up, down, expert_begin: int = 0, out=None):
    """The expert layer of a few tokens over 4-bit weights: gate_up = (packed [L,2I,H/2], scales, zeros), down = (packed [L,H,I/2],
    scales, zeros).  Returns [T,H] in x's type; slots whose expert is not local do not count."""
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x must be a BF16 or FP16 tensor")
    _require("x", x, x.dtype)
    dev = x.device
    first = _w4("gate_up", *gate_up, x.dtype, dev, 3)
    second = _w4("down", *down, x.dtype, dev, 3)
    local = gate_up[0].shape[0]
    if down[0].shape[0] != local or first.n != 2 * second.k or first.k != second.n:
        raise ValueError("gate_up [L, 2I, H/2] and down [L, H, I/2] do not belong together")
    if x.ndim != 2 or x.shape[1] != first.k:
        raise ValueError(f"x must be [T, {first.k}] (got {tuple(x.shape)})")
    tokens = x.shape[0]
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("topk_idx must be an int64 or int32 tensor")
    _require("topk_idx", topk_idx, topk_idx.dtype, device=dev)
    if topk_idx.ndim != 2 or topk_idx.shape[0] != tokens or topk_idx.shape[1] == 0:
        raise ValueError("topk_idx must be [T, K]")
    topk = topk_idx.shape[1]
    _require("topk_weights", topk_weights, torch.float32, (tokens, topk), dev)
    _at_most(_MAX_TOPK, topk=topk)
    _at_most(_W4_MAX_ROUTES, routes=tokens * topk)
    _at_most(_MAX_LOCAL_EXPERTS, experts=local)
    try:
        begin = operator.index(expert_begin)
    except TypeError:
        begin = -1
    if not 0 <= begin < 1 << 31:
        raise ValueError("expert_begin must be an integer in [0, 2^31)")
    if out is None:
        out = torch.empty((tokens, first.k), dtype=x.dtype, device=dev)
    else:
        _require("out", out, x.dtype, (tokens, first.k), dev)
    lib = _lib.load()
    x = _aligned(x)
    scratch = torch.empty((lib.dpep_w4_experts_scratch_bytes(tokens, topk, first.k, second.k),), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        status = lib.dpep_w4_experts(ctypes.byref(first), ctypes.byref(second), _TYPES[x.dtype], _ptr(x), _ptr(topk_idx), topk_idx.element_size(),
                                     _ptr(topk_weights), tokens, topk, begin, local, _ptr(out), _ptr(scratch), _stream(dev))
    _lib.check(status, "w4_experts")
    return out


# ---------------------------------------------------------------------------------------------
# Norm, dense gated block, products in 8-bit integers
# ---------------------------------------------------------------------------------------------
_NORM_MAX_HIDDEN, _NORM_MAX_TOKENS = 16384, 0x7FFFFF
_FFN_MAX_DIM, _FFN_MAX_TOKENS = 65536, 0x1FFFFF
_W8_MAX_K, _W8_MAX_N, _W8_MAX_ROWS = 65536, 0x1FFFFF, 0x1FFFFF
QUANTIZE = {None: (0, 8), "fp8": (1, 16), "mxfp8": (2, 32), "int8": (3, 16)}  # DPEP_QUANT_*, what H is a multiple of


class _Norm(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("x", "residual", "weight", "stream_out", "y", "rstd", "codes", "scales")] + [
        ("eps", ctypes.c_float)] + [(name, ctypes.c_int32) for name in ("type", "weight_type", "quantize", "num_tokens", "hidden")]


class _NormGradients(ctypes.Structure):
    _fields_ = [(name, ctypes.c_void_p) for name in ("grad_y", "stream", "weight", "rstd", "grad_stream", "grad_x", "grad_weight")] + [
        (name, ctypes.c_int32) for name in ("type", "weight_type", "num_tokens", "hidden")]


class _Ffn(ctypes.Structure):
    _fields_ = [("gate_up", ctypes.c_void_p), ("down", ctypes.c_void_p), ("type", ctypes.c_int32), ("hidden", ctypes.c_int32), ("inter", ctypes.c_int32)]


class _W8(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("n", ctypes.c_int32), ("k", ctypes.c_int32)]


def _address(t):
    return None if t is None else t.data_ptr()


def _require_rows(name, x, types, unit, most, most_rows):
    """x as rows [T,H] of one of `types`, H a multiple of `unit` up to `most`."""
    if not isinstance(x, torch.Tensor) or x.dtype not in types:
        raise ValueError(f"{name} must be a tensor of " + ", ".join(str(t) for t in types))
    _require(name, x, x.dtype)
    if x.ndim != 2 or x.shape[1] == 0 or x.shape[1] % unit or x.shape[1] > most:
        raise ValueError(f"{name} must be [rows, width], its width a multiple of {unit} up to {most} (got {tuple(x.shape)})")
    _at_most(most_rows, rows=x.shape[0])
    return x.shape


def _require_norm_weight(weight, x):
    if not isinstance(weight, torch.Tensor) or weight.dtype not in (x.dtype, torch.float32):
        raise ValueError("weight must be a tensor of x's type or FP32")
    _require("weight", weight, weight.dtype, (x.shape[1],), x.device)


def rms_norm(x, weight, residual=None, eps: float = 1e-6, quantize=None, output: bool = True):
    """(y or None, stream or None without a residual, rstd, codes or None, scales or None)."""
    if quantize not in QUANTIZE:
        raise ValueError(f"quantize must be one of {sorted(name for name in QUANTIZE if name)} or None")
    code, unit = QUANTIZE[quantize]
    tokens, hidden = _require_rows("x", x, tuple(_TYPES), unit, _NORM_MAX_HIDDEN, _NORM_MAX_TOKENS)
    _require_norm_weight(weight, x)
    if residual is not None:
        _require("residual", residual, x.dtype, tuple(x.shape), x.device)
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0 <= eps <= 1:
        raise ValueError("eps must be a number in [0, 1]")
    if not output and quantize is None:
        raise ValueError("output=False leaves nothing without quantize")
    dev = x.device
    y = torch.empty_like(x) if output else None
    stream = None if residual is None else torch.empty_like(x)
    rstd = torch.empty((tokens,), dtype=torch.float32, device=dev)
    codes = scales = None
    if quantize == "fp8":
        codes = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty((tokens, (hidden + 127) // 128), dtype=torch.float32, device=dev)
    elif quantize == "mxfp8":
        codes = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty((tokens, hidden // 32), dtype=torch.uint8, device=dev)
    elif quantize == "int8":
        codes = torch.empty((tokens, hidden), dtype=torch.int8, device=dev)
        scales = torch.empty((tokens,), dtype=torch.float32, device=dev)
    x, weight, residual = _aligned(x), _aligned(weight), None if residual is None else _aligned(residual)
    call = _Norm(_address(x), _address(residual), _address(weight), _address(stream), _address(y), _address(rstd), _address(codes), _address(scales),
                 float(eps), _TYPES[x.dtype], _TYPES[weight.dtype], code, tokens, hidden)
    with _on_device(dev):
        status = _lib.load().dpep_rms_norm(ctypes.byref(call), _stream(dev))
    _lib.check(status, "rms_norm")
    return y, stream, rstd, codes, scales


def rms_norm_backward(grad_y, stream, weight, rstd, grad_stream=None):
    """(grad_x in the rows' type, grad_weight FP32 [H])."""
    tokens, hidden = _require_rows("stream", stream, tuple(_TYPES), 8, _NORM_MAX_HIDDEN, _NORM_MAX_TOKENS)
    dev = stream.device
    _require("grad_y", grad_y, stream.dtype, (tokens, hidden), dev)
    _require_norm_weight(weight, stream)
    _require("rstd", rstd, torch.float32, (tokens,), dev)
    if grad_stream is not None:
        _require("grad_stream", grad_stream, stream.dtype, (tokens, hidden), dev)
    lib = _lib.load()
    grad_x = torch.empty_like(stream)
    grad_weight = torch.empty((hidden,), dtype=torch.float32, device=dev)
    scratch = torch.empty((lib.dpep_rms_norm_backward_scratch_bytes(tokens, hidden),), dtype=torch.uint8, device=dev)
    grad_y, stream, weight, grad_stream = _aligned(grad_y), _aligned(stream), _aligned(weight), None if grad_stream is None else _aligned(grad_stream)
    call = _NormGradients(_address(grad_y), _address(stream), _address(weight), _address(rstd), _address(grad_stream), _address(grad_x), _address(grad_weight),
                          _TYPES[stream.dtype], _TYPES[weight.dtype], tokens, hidden)
    with _on_device(dev):
        status = lib.dpep_rms_norm_backward(ctypes.byref(call), _ptr(scratch), _stream(dev))
    _lib.check(status, "rms_norm_backward")
    return grad_x, grad_weight


def _ffn(x, gate_up, down):
    """Sizes of a gated block after its checks: (tokens, hidden, inter)."""
    tokens, hidden = _require_rows("x", x, (torch.bfloat16, torch.float16), 8, _FFN_MAX_DIM, _FFN_MAX_TOKENS)
    if not isinstance(down, torch.Tensor) or down.ndim != 2 or down.shape[0] != hidden or down.shape[1] == 0 or down.shape[1] % 8 or down.shape[1] > _FFN_MAX_DIM:
        raise ValueError(f"down must be [{hidden}, I], I a multiple of 8 up to {_FFN_MAX_DIM}")
    inter = down.shape[1]
    _require("gate_up", gate_up, x.dtype, (2 * inter, hidden), x.device)
    _require("down", down, x.dtype, None, x.device)
    return tokens, hidden, inter


def gated_ffn(x, gate_up, down, keep: bool = False):
    """y [T,H], or (y, kept FP32 [T,2I])."""
    tokens, hidden, inter = _ffn(x, gate_up, down)
    dev, lib = x.device, _lib.load()
    y = torch.empty_like(x)
    kept = torch.empty((tokens, 2 * inter), dtype=torch.float32, device=dev) if keep else None
    scratch = torch.empty((lib.dpep_gated_ffn_scratch_bytes(tokens, hidden, inter),), dtype=torch.uint8, device=dev)
    x, gate_up, down = _aligned(x), _aligned(gate_up), _aligned(down)
    call = _Ffn(_address(gate_up), _address(down), _TYPES[x.dtype], hidden, inter)
    with _on_device(dev):
        status = lib.dpep_gated_ffn(ctypes.byref(call), _ptr(x), tokens, _ptr(y), _ptr(kept), _ptr(scratch), _stream(dev))
    _lib.check(status, "gated_ffn")
    return (y, kept) if keep else y


def gated_ffn_backward(grad_y, x, gate_up, down, kept):
    """(grad_x, grad_gate_up, grad_down) in x's type."""
    tokens, hidden, inter = _ffn(x, gate_up, down)
    dev, lib = x.device, _lib.load()
    _require("grad_y", grad_y, x.dtype, (tokens, hidden), dev)
    _require("kept", kept, torch.float32, (tokens, 2 * inter), dev)
    grad_x, grad_gate_up, grad_down = torch.empty_like(x), torch.empty_like(gate_up), torch.empty_like(down)
    scratch = torch.empty((lib.dpep_gated_ffn_backward_scratch_bytes(tokens, hidden, inter),), dtype=torch.uint8, device=dev)
    grad_y, x, gate_up, down, kept = (_aligned(t) for t in (grad_y, x, gate_up, down, kept))
    call = _Ffn(_address(gate_up), _address(down), _TYPES[x.dtype], hidden, inter)
    with _on_device(dev):
        status = lib.dpep_gated_ffn_backward(ctypes.byref(call), _ptr(grad_y), _ptr(x), _ptr(kept), tokens, _ptr(grad_x), _ptr(grad_gate_up), _ptr(grad_down),
                                             _ptr(scratch), _stream(dev))
    _lib.check(status, "gated_ffn_backward")
    return grad_x, grad_gate_up, grad_down


def quantize_tokens(x):
    """(codes int8 [T,K], scales FP32 [T])."""
    tokens, k = _require_rows("x", x, tuple(_TYPES), 16, _W8_MAX_K, _W8_MAX_ROWS)
    codes = torch.empty((tokens, k), dtype=torch.int8, device=x.device)
    scales = torch.empty((tokens,), dtype=torch.float32, device=x.device)
    x = _aligned(x)
    with _on_device(x.device):
        status = _lib.load().dpep_quantize_tokens(_ptr(x), _TYPES[x.dtype], tokens, k, _ptr(codes), _ptr(scales), _stream(x.device))
    _lib.check(status, "quantize_tokens")
    return codes, scales


def w8_matmul(x, codes, scales, dtype=None):
    """x [T,K], or (codes int8 [T,K], scales FP32 [T]), times (codes int8 [N,K], scales FP32 [N]): [T,N] in `dtype`."""
    if dtype is not None and dtype not in _TYPES:
        raise ValueError("dtype must be FP32, BF16 or FP16")
    n, k = _require_rows("codes", codes, (torch.int8,), 16, _W8_MAX_K, _W8_MAX_N)
    if n == 0:
        raise ValueError("codes must have a row")
    dev = codes.device
    _require("scales", scales, torch.float32, (n,), dev)
    if isinstance(x, (tuple, list)):
        if len(x) != 2:
            raise ValueError("x must be a tensor or a pair of codes and scales")
        rows, rows_k = _require_rows("x codes", x[0], (torch.int8,), 16, _W8_MAX_K, _W8_MAX_ROWS)
        _require("x codes", x[0], torch.int8, None, dev)
        _require("x scales", x[1], torch.float32, (rows,), dev)
        dtype = torch.bfloat16 if dtype is None else dtype
    else:
        rows, rows_k = _require_rows("x", x, tuple(_TYPES), 16, _W8_MAX_K, _W8_MAX_ROWS)
        _require("x", x, x.dtype, None, dev)
        dtype = x.dtype if dtype is None else dtype
    if rows_k != k:
        raise ValueError(f"x must be [T, {k}] (got [{rows}, {rows_k}])")
    x_codes, x_scales = x if isinstance(x, (tuple, list)) else quantize_tokens(x)
    lib = _lib.load()
    y = torch.empty((rows, n), dtype=dtype, device=dev)
    scratch = torch.empty((lib.dpep_w8_matmul_scratch_bytes(rows, n, k),), dtype=torch.uint8, device=dev)
    x_codes, codes = _aligned(x_codes), _aligned(codes)
    call = _W8(_address(codes), _address(scales), n, k)
    with _on_device(dev):
        status = lib.dpep_w8_matmul(ctypes.byref(call), _ptr(x_codes), _ptr(x_scales), rows, _TYPES[dtype], _ptr(y), _ptr(scratch), _stream(dev))
    _lib.check(status, "w8_matmul")
    return y


class _ProductChoice(ctypes.Structure):
    _fields_ = [(name, ctypes.c_int32) for name in ("way", "parts", "stream_groups", "stream_blocks", "stream_stages", "together")] + [("workgroups", ctypes.c_int64)]


PRODUCT_WAYS = ("stream", "ring", "pairs", "large")
_PRODUCTS = {"ffn": 0, "ffn_backward": 1, "w8": 2}  # DPEP_PRODUCTS_*


def product_choices(operation: str, rows: int, a: int, b: int):
    """How calls of these sizes make their products: dicts of ``way`` (of ``PRODUCT_WAYS``), ``parts`` of k, ``stream`` (groups, blocks, stages; or None), ``together`` and
    ``workgroups``.  ``operation``: ``"ffn"`` (rows, H, I: gate and up, then down), ``"ffn_backward"`` (dh, then the gradients of x, gate_up and down) or ``"w8"`` (rows, N, K).  Host arithmetic only."""
    made = (_ProductChoice * 4)()
    count = _lib.load().dpep_product_choices(_PRODUCTS[operation], rows, a, b, made)
    _lib.check(min(count, 0), "product_choices")
    return [dict(way=PRODUCT_WAYS[c.way], parts=c.parts, stream=(c.stream_groups, c.stream_blocks, c.stream_stages) if c.way == 0 else None, together=bool(c.together),
                 workgroups=c.workgroups) for c in made[:count]]
