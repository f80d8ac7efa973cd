"""4-bit products in 64 bits, with a bound on what fp32 sums may be off by.  Test infrastructure only."""

from __future__ import annotations

import numpy as np

# An fp32 sum of products (q + 16) x over a group, of which (zero + 16) times the sum of x is taken again, is off by at most a few
# roundings of its largest partial sum: 2^-24 * 32 * sum |x| * scale each; 2^-18 leaves room for a group's worth of them in sequence.
SUM_SLACK = 2.0**-18


def unpack(packed, scales, zeros=None):
    """Values [..., N, K] and their groups' scales, one for each value."""
    packed = np.asarray(packed, dtype=np.int64)
    q = np.empty((*packed.shape[:-1], packed.shape[-1] * 2))
    q[..., 0::2], q[..., 1::2] = packed & 15, packed >> 4
    group = q.shape[-1] // scales.shape[-1]
    wide = np.repeat(np.asarray(scales, dtype=np.float64), group, axis=-1)
    shift = 8.0 if zeros is None else np.repeat(np.asarray(zeros, dtype=np.float64), group, axis=-1)
    return (q - shift) * wide, np.abs(wide)


def product(x, weights):
    """(y [M,N], bound [M,N]) of x [M,K] and one matrix."""
    w, scale = unpack(*weights)
    return x @ w.T, SUM_SLACK * 32 * np.abs(x) @ scale.T


def experts(x, ids, route_weights, gate_up, down, begin=0):
    """(y [T,H], bound [T,H]); ids outside [begin, begin + L) do not count."""
    tokens, hidden = x.shape
    y, bound = np.zeros((tokens, hidden)), np.zeros((tokens, hidden))
    local = gate_up[0].shape[0]

    def of(weights, e):
        return [None if part is None else part[e] for part in weights]

    for t in range(tokens):
        for s, raw in enumerate(ids[t]):
            e = int(raw) - begin
            if not 0 <= e < local:
                continue
            both, off = product(x[t : t + 1], of(gate_up, e))
            inter = both.shape[1] // 2
            g, u = both[0, :inter], both[0, inter:]
            sig = 1.0 / (1.0 + np.exp(-g))
            h = g * sig * u
            # h is held in 16 bits of mantissa; its inputs' bounds go through silu (slope at most 1.1) and the product
            h_off = 2.0**-16 * np.abs(h) + 1.1 * off[0, :inter] * np.abs(u) + off[0, inter:] * np.abs(g * sig)
            w2, scale = unpack(*of(down, e))
            y[t] += route_weights[t, s] * (w2 @ h)
            bound[t] += np.abs(route_weights[t, s]) * (np.abs(w2) @ h_off + SUM_SLACK * 32 * scale @ np.abs(h))
    return y, bound


def sum_deviation(x, weights):
    """Standard deviation [M,N] of what 32-bit sums of x [M,K] with one matrix are off by, none of them smaller: in a group of G values no partial sum is
    larger than 64 sum |x| (a code counts as 16 to 31, and the group's sum times as much is taken off), so a rounding has at most
    2^-24 of that, evenly spread; 2 G of them, and one for every group in the sum over groups."""
    _, scale = unpack(*weights)
    groups = np.asarray(weights[1]).shape[-1]
    group = scale.shape[-1] // groups
    largest = 64 * np.abs(x).reshape(len(x), groups, group).sum(axis=-1)  # [M, groups]
    each = 2.0**-24 / np.sqrt(3) * largest
    scale = scale[:, ::group]
    return np.sqrt((2 * group + groups) * (each**2 @ (scale**2).T))


def bf16(v):
    """Values rounded to BF16 (to nearest, ties to even)."""
    bits = np.asarray(v, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)


def experts_and_deviation(x, ids, route_weights, gate_up, down, hold=lambda h: h):
    """(y [T,H], deviation [T,H]) where the rows between the products are held to 16 bits of mantissa (off by at most 2^-16 of
    themselves, evenly spread), for ids 0 .. L-1 or -1.  hold: what becomes of these rows instead, in a test of the deviation itself."""
    tokens, hidden = x.shape
    y, variance = np.zeros((tokens, hidden)), np.zeros((tokens, hidden))

    def of(weights, e):
        return [None if part is None else part[e] for part in weights]

    for t in range(tokens):
        for s, e in enumerate(ids[t]):
            if e < 0:
                continue
            first = of(gate_up, e)
            both, off = product(x[t : t + 1], first)[0][0], sum_deviation(x[t : t + 1], first)[0]
            inter = len(both) // 2
            g, u = both[:inter], both[inter:]
            sig = 1.0 / (1.0 + np.exp(-g))
            h = route_weights[t, s] * g * sig * u
            # silu's slope is at most 1.1
            h_variance = h**2 * 4.0**-16 / 3 + route_weights[t, s] ** 2 * ((1.1 * off[:inter] * u) ** 2 + (off[inter:] * g * sig) ** 2)
            second = of(down, e)
            w2, _ = unpack(*second)
            y[t] += w2 @ hold(h)
            variance[t] += w2**2 @ h_variance + sum_deviation(h[None], second)[0] ** 2
    return y, np.sqrt(variance)
