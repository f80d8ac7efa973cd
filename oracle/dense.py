"""Norm, gated feed-forward block and products in 8-bit integers in 64 bits, with bounds on what 32-bit arithmetic and the roundings to fewer
bits may be off by.  Test infrastructure only."""

from __future__ import annotations

import numpy as np

EPS32 = 2.0**-24  # half a step of fp32, relative
HALF = {"bf16": 2.0**-8, "fp16": 2.0**-11, "fp32": 2.0**-24}  # half a step of a type, relative
TINY = {"bf16": 0.0, "fp16": 2.0**-25, "fp32": 0.0}  # and absolute, where values are subnormal (fp16 alone gets there)
# A row of up to 16384 squares is summed 64 in sequence by a thread, then in trees and over 16 waves: under 128 roundings; the root,
# quotient and products behind it are a few more.
NORM_SLACK = 128 * EPS32


def norm(s, weight, eps):
    """(v, rstd) of rows s [T,H]."""
    rstd = 1.0 / np.sqrt((s * s).mean(axis=1) + eps)
    return s * rstd[:, None] * weight, rstd


def norm_backward(g, s, weight, eps, grad_stream=None):
    """(grad_x, its bound before the last rounding, grad_weight, its bound)."""
    _, rstd = norm(s, weight, eps)
    hat = s * rstd[:, None]
    gw = g * weight
    mean = (gw * hat).mean(axis=1, keepdims=True)
    grad = rstd[:, None] * (gw - hat * mean)
    size = rstd[:, None] * (np.abs(gw) + np.abs(hat) * np.abs(gw * hat).mean(axis=1, keepdims=True))
    if grad_stream is not None:
        grad, size = grad + grad_stream, size + np.abs(grad_stream)
    each = np.abs(g * hat).sum(axis=0)
    # (a column is summed over the rows of a workgroup, of which there are 256 to 1024 if there are as many rows, then over those: 64 at a time)
    return grad, 4 * NORM_SLACK * size, (g * hat).sum(axis=0), (NORM_SLACK + (len(s) / 256 + 64) * EPS32) * each


def fp8_blocks(v):
    """(what each code stands for before it is rounded [T,H], scales [T,ceil(H/128)])."""
    blocks = [v[:, at : at + 128] for at in range(0, v.shape[1], 128)]
    largest = np.stack([np.maximum(np.abs(b).max(axis=1), 1e-4) for b in blocks], axis=1)
    wide = np.repeat(largest, 128, axis=1)[:, : v.shape[1]]
    return v * 448.0 / wide, largest / 448.0


def e4m3_bound(target):
    """Half a step of e4m3 around each number."""
    return np.maximum(2.0**-4 * np.abs(target), 2.0**-10)


def tokens(v):
    """(what each 8-bit integer stands for before it is rounded, scales [T])."""
    largest = np.maximum(np.abs(v).max(axis=1), 1e-20)
    return v * (127.0 / largest)[:, None], largest / 127.0


def _sum_bound(k, size):
    """What a sum of k products in fp32 may be off by: the matrix cores add 32 at a time (each of them rounded at most once on its way) to a running sum."""
    return EPS32 * (k / 16 + 48) * size


def _silu(g):
    share = 1.0 / (1.0 + np.exp(-g))
    return g * share, share


def _share_off(g, share):
    """What the share may be off by in 32 bits, as 1 / (1 + 2^(-g log2 e)) with a power and a reciprocal that are good to a whole step (2 half steps, relative): the power's argument
    is off by the half step of its product and 0.224 of one of the constant, 1.23 |g| half steps of the power, and the power by 2 more; these count by the power's share (1 - share)
    of the sum, which is rounded once; the reciprocal 2.  What falls below 2^-126 may be lost."""
    return ((1.23 * np.abs(g) + 2.0) * (1.0 - share) + 3.0) * EPS32 * share + 2.0**-126


def h_off(g, u):
    """What h = (g share) u may be off by in 32 bits, g and u exact: the share's, and two products."""
    silu, share = _silu(g)
    return np.abs(g * u) * _share_off(g, share) + 2 * EPS32 * np.abs(silu * u)


def dz_off(dh, g, u):
    """The same of dg = ((dh u) share) (1 + g (1 - share)) and du = (dh g) share: with w = 1 + q, q = g (1 - share), the share's where it is a factor, and three products; w's, which are
    |g| times the share's, the rounding of 1 - share and of q, and that of the sum."""
    silu, share = _silu(g)
    q = g * (1.0 - share)
    off, w = _share_off(g, share), np.abs(1.0 + q)
    dg = np.abs(dh * u) * (w * (off + 3 * EPS32 * share) + (share + off) * (np.abs(g) * off + 2 * EPS32 * np.abs(q) + EPS32 * w))
    return dg, np.abs(dh * g) * off + 2 * EPS32 * np.abs(dh * silu)


def ffn(x, gate_up, down, dtype):
    """dict of y, its bound, and what a backward pass needs of the intermediate values."""
    inter = down.shape[1]
    z = x @ gate_up.T
    z_off = _sum_bound(x.shape[1], np.abs(x) @ np.abs(gate_up).T)
    g, u, g_off, u_off = z[:, :inter], z[:, inter:], z_off[:, :inter], z_off[:, inter:]
    silu, share = _silu(g)
    h = silu * u
    # silu's slope is at most 1.1
    off = 1.1 * g_off * (np.abs(u) + u_off) + np.abs(silu) * u_off + h_off(g, u)
    off = off + HALF[dtype] * (np.abs(h) + off) + TINY[dtype]
    y = h @ down.T
    y_off = off @ np.abs(down).T + _sum_bound(inter, (np.abs(h) + off) @ np.abs(down).T)
    return dict(y=y, y_off=y_off + HALF[dtype] * (np.abs(y) + y_off) + TINY[dtype], z=z, z_off=z_off, g=g, u=u, g_off=g_off, u_off=u_off, h=h, h_off=off, silu=silu,
                share=share)


def ffn_backward(grad_y, x, gate_up, down, dtype):
    """[(gradient, bound)] of x, gate_up and down."""
    f = ffn(x, gate_up, down, dtype)
    dh = grad_y @ down
    dh_off = _sum_bound(grad_y.shape[1], np.abs(grad_y) @ np.abs(down))
    slope = f["share"] * (1.0 + f["g"] * (1.0 - f["share"]))
    dg, du = dh * f["u"] * slope, dh * f["silu"]
    size, u_size = np.abs(dh) + dh_off, np.abs(f["u"]) + f["u_off"]
    # silu's slope is at most 1.1 and its change at most 0.5
    own = dz_off(size, f["g"], u_size)
    dg_off = 1.1 * (dh_off * u_size + size * f["u_off"]) + 0.5 * size * u_size * f["g_off"] + own[0]
    du_off = dh_off * np.abs(f["silu"]) + 1.1 * size * f["g_off"] + own[1]
    dz, off = np.concatenate([dg, du], axis=1), np.concatenate([dg_off, du_off], axis=1)
    off = off + HALF[dtype] * (np.abs(dz) + off) + TINY[dtype]

    def product(a, b, a_off, b_off, k):
        value, size = a @ b, (np.abs(a) + a_off) @ (np.abs(b) + b_off)
        all_off = size - np.abs(a) @ np.abs(b) + _sum_bound(k, size)
        return value, all_off + HALF[dtype] * (np.abs(value) + all_off) + TINY[dtype]

    zero = 0.0
    return [product(dz, gate_up, off, zero, dz.shape[1]), product(dz.T, x, off.T, zero, len(x)), product(grad_y.T, f["h"], zero, f["h_off"], len(x))]
