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
