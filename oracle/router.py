"""Router and balance loss in 64 bits, by their definitions, one token at a time; gradients by the formulas and by differences.

Test infrastructure only.  Keys are rounded to fp32 as the operator defines them, everything else stays in float64.
"""

from __future__ import annotations

import numpy as np

NEG = -np.inf


def sigmoid(z):
    z = np.asarray(z, dtype=np.float64)
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def choose(z, topk, score="softmax", bias=None, real=True, groups=1, topk_groups=1):
    """Expert ids of one token's logits (float64 [E]), best first, -1 where none is left."""
    experts = len(z)
    if score == "softmax":
        keys = np.asarray(z, dtype=np.float32).copy()
    else:
        keys = sigmoid(z).astype(np.float32)
        if bias is not None:
            keys = (keys + np.asarray(bias, dtype=np.float32)).astype(np.float32)
    keys[np.isnan(keys)] = np.inf
    keys[np.asarray(z) == NEG] = NEG
    if not real:
        keys[:] = NEG
    if groups > 1:
        width = experts // groups
        value = []
        for g in range(groups):
            best = sorted(keys[g * width : (g + 1) * width], reverse=True)
            two = score == "sigmoid" and width > 1 and best[1] != NEG
            value.append(np.float32(best[0] + best[1]) if two else best[0])
        order = sorted(range(groups), key=lambda g: (-value[g], g))
        for g in order[topk_groups:]:
            keys[g * width : (g + 1) * width] = NEG
    order = sorted(range(experts), key=lambda e: (-keys[e], e))[:topk]
    return [e if keys[e] != NEG else -1 for e in order]


def weights_of(z, ids, score="softmax", normalize=True, scale=1.0):
    """Route weights [K] of one token (float64)."""
    z = np.asarray(z, dtype=np.float64)
    ids = np.asarray(ids)
    found = ids >= 0
    out = np.zeros(len(ids))
    if not found.any():
        return out
    picked = z[ids[found]]
    if score == "sigmoid":
        s = sigmoid(picked)
        out[found] = s / (s.sum() + 1e-20) if normalize else s
    else:
        over = picked if normalize else z
        top = over.max()
        out[found] = np.exp(picked - top) / np.exp(over - top).sum()
    return out * scale


def probabilities(z, score):
    """p of the balance loss for one token."""
    z = np.asarray(z, dtype=np.float64)
    if score == "sigmoid":
        s = sigmoid(z)
        return s / (s.sum() + 1e-20)
    if (z == NEG).all():
        return np.zeros(len(z))
    e = np.exp(z - z.max())
    return e / e.sum()


def balance(z, ids, score="softmax", offsets=None):
    """(losses [B], counts [B,E], tokens [B]) of logits [T,E] and ids [T,K]."""
    tokens, experts = z.shape
    bounds = [0, tokens] if offsets is None else list(offsets)
    losses, counts, members = [], [], []
    for begin, end in zip(bounds[:-1], bounds[1:]):
        count, mean, held = np.zeros(experts, dtype=np.int64), np.zeros(experts), 0
        for t in range(begin, end):
            routes = [e for e in ids[t] if e >= 0]
            if not routes:
                continue
            held += 1
            for e in routes:
                count[e] += 1
            mean += probabilities(z[t], score)
        losses.append((mean / held * count * experts / count.sum()).sum() if held else 0.0)
        counts.append(count)
        members.append(held)
    return np.array(losses), np.array(counts), np.array(members)


def weights_gradient(z, ids, g, score="softmax", normalize=True, scale=1.0):
    """d (sum_k g_k w_k) / dz for one token, by the chain rule over the whole Jacobian of the weights."""
    z = np.asarray(z, dtype=np.float64)
    grad = np.zeros(len(z))
    found = [k for k, e in enumerate(ids) if e >= 0]
    if not found:
        return grad
    e = np.array([ids[k] for k in found])
    up = np.array([g[k] for k in found], dtype=np.float64) * scale
    if score == "sigmoid":
        s = sigmoid(z[e])
        slope = s * sigmoid(-z[e])
        total = s.sum() + 1e-20
        jacobian = np.diag(slope / total) - np.outer(s, slope) / total**2 if normalize else np.diag(slope)
        grad[e] = up @ jacobian
    elif normalize:
        p = np.exp(z[e] - z[e].max())
        p /= p.sum()
        grad[e] = up @ (np.diag(p) - np.outer(p, p))
    else:
        p = probabilities(z, "softmax")
        grad = up @ (np.eye(len(z))[e] * p - np.outer(p[e], p))
    return grad


def balance_gradient(z, ids, grad_losses, score="softmax", offsets=None):
    """d (sum_b g_b loss_b) / dz, [T,E]."""
    tokens, experts = z.shape
    bounds = [0, tokens] if offsets is None else list(offsets)
    _, counts, members = balance(z, ids, score, offsets)
    grad = np.zeros((tokens, experts))
    for b, (begin, end) in enumerate(zip(bounds[:-1], bounds[1:])):
        for t in range(begin, end):
            if not any(e >= 0 for e in ids[t]):
                continue
            up = grad_losses[b] / members[b] * counts[b] * experts / counts[b].sum()  # dL/dp
            p = probabilities(z[t], score)
            if score == "softmax":
                grad[t] = p * (up - (up * p).sum())
            else:
                s = sigmoid(z[t])
                grad[t] = s * sigmoid(-z[t]) / (s.sum() + 1e-20) * (up - (up * p).sum())
    return grad
