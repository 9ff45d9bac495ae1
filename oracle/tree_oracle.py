"""CPU oracle for generation over drafted trees and for distillation, in 64 bits.

TEST INFRASTRUCTURE ONLY, as the other oracles: written from the definitions in
``include/mt_attention.h`` and ``include/mt_ops.h``, node by node.  Where a test
needs a bound on the rounding errors of the fp32 / 16-bit operator, the function
returns the sums that the bound is made of.  Pinned in tests/test_tree_oracle.py
against torch in float64, closed forms and the distribution that the
verification has to leave unchanged.
"""

from __future__ import annotations

import numpy as np

LOW, HIGH = float(np.finfo(np.float32).min), float(np.finfo(np.float32).max)


def ancestors(parents):
    """Per node the list of its ancestors and itself, root first; None for padding."""
    out = []
    for n, p in enumerate(parents):
        if p == -1:
            out.append([n])
        elif 0 <= p < n and out[p] is not None:
            out.append(out[p] + [n])
        else:
            out.append(None)
    return out


def tree_rope(x, cos, sin, length, parents):
    """x [H, N, D] of one sequence, tables [rows, D/2]: (rotated, sum of the products' magnitudes)."""
    y, mag = np.zeros(x.shape), np.zeros(x.shape)
    for n, up in enumerate(ancestors(parents)):
        if up is None:
            continue
        pos = min(length + len(up) - 1, len(cos) - 1)
        e, o, c, s = x[:, n, 0::2], x[:, n, 1::2], cos[pos], sin[pos]
        y[:, n, 0::2], y[:, n, 1::2] = e * c - o * s, e * s + o * c
        mag[:, n, 0::2], mag[:, n, 1::2] = abs(e * c) + abs(o * s), abs(e * s) + abs(o * c)
    return y, mag


def tree_attention(q, k, v, kc, vc, length, parents, scale):
    """One sequence: q [Hq, N, D], k / v [Hkv, N, D], caches [Hkv, cap, D].
    Returns (out, sum_j p_j |v_j|, the largest sum_d |q_d k_d| scale over the keys seen)."""
    hq, n_nodes, d = q.shape
    hkv = k.shape[0]
    r = hq // hkv
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for n, up in enumerate(ancestors(parents)):
        if up is None:
            continue
        for g in range(hkv):
            keys = np.concatenate((kc[g, :length], k[g, up]))
            vals = np.concatenate((vc[g, :length], v[g, up]))
            qs = q[g * r:(g + 1) * r, n]
            s = qs @ keys.T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[g * r:(g + 1) * r, n] = p @ vals
            mag[g * r:(g + 1) * r, n] = p @ abs(vals)
            top[g * r:(g + 1) * r, n] = (abs(qs) @ abs(keys).T * scale).max(-1)
    return out, mag, top


def top_softmax(x, k):
    x = np.clip(np.where(np.isnan(x), LOW, x), LOW, HIGH).astype(np.float64)
    kept = x >= np.sort(x)[-k]
    with np.errstate(over="ignore"):
        w = np.where(kept, np.exp(x - x.max()), 0.0)
    return w / w.sum()


def topk_verify(logits, tokens, parents, uniform, noise, k, draft=None):
    """One sequence: (path, token)."""
    if parents[0] != -1:
        return [], 0
    path = [0]
    while True:
        u = path[-1]
        p = top_softmax(logits[u], k)
        kids = [c for c in range(u + 1, len(parents)) if parents[c] == u]
        taken = None
        for c in kids:
            x = tokens[c]
            inside = 0 <= x < p.size
            q = np.zeros(p.size) if draft is None else top_softmax(draft[u], k)
            if draft is None and inside:
                q[x] = 1.0
            if inside and float(uniform[c]) * q[x] < p[x]:
                taken = c
                break
            left = np.maximum(p - q, 0.0)
            if left.sum() > 0:
                p = left / left.sum()
        if taken is None:
            with np.errstate(divide="ignore"):
                score = np.where(p > 0, p / noise.astype(np.float64), -1.0)
            return path, int(score.argmax())
        path.append(taken)


def distillation(logits, teacher, index, temperature):
    """(loss, gradient, error terms): rows [R, V] and [R, K] in float64.  The error
    terms are q, P and sum_j p_j (1 + |log p_j| + |log q_j|) a row, with the count."""
    t = float(temperature)
    rows, vocab = logits.shape
    grad, q_all, p_all = (np.zeros((rows, vocab)) for _ in range(3))
    terms = np.zeros(rows)
    loss, count = 0.0, 0
    for r in range(rows):
        use = (index[r] >= 0) & (teacher[r] > -np.inf)
        if not use.any():
            continue
        count += 1
        y = teacher[r][use] / t
        p = np.exp(y - y.max())
        p /= p.sum()
        x = logits[r] / t
        logq = x - x.max() - np.log(np.exp(x - x.max()).sum())
        logp, at = np.log(p), index[r][use]
        with np.errstate(invalid="ignore"):
            loss += float(np.where(p > 0, p * (logp - logq[at]), 0.0).sum())
        np.add.at(p_all[r], at, p)
        q_all[r] = np.exp(logq)
        grad[r] = q_all[r] - p_all[r]
        terms[r] = float((p * (1 + abs(logp) + abs(logq[at]))).sum())
    n = max(count, 1)
    return loss * t * t / n, grad * (t / n), dict(q=q_all, p=p_all, terms=terms, count=count)
