"""Plain forms in 64 bits of the operators whose rows choose their weights, and seeded cases of them."""
from __future__ import annotations

import numpy as np

GELU_C = 0.7978845608028654


def gelu(x):
    return 0.5 * x * (1 + np.tanh(GELU_C * (x + 0.044715 * x ** 3)))


def gelu_grad(x):
    t = np.tanh(GELU_C * (x + 0.044715 * x ** 3))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * GELU_C * (1 + 3 * 0.044715 * x * x)


def choose(logits, k):
    """ids [T, k]: the k largest above -infinity, the lower index first among equals, NaN largest; -1 where none."""
    T, E = logits.shape
    x = np.where(np.isnan(logits), np.inf, logits.astype(np.float64))
    nan = np.isnan(logits)
    ids = np.full((T, k), -1, np.int32)
    for t in range(T):
        order = sorted((e for e in range(E) if x[t, e] != -np.inf), key=lambda e: (not nan[t, e], -x[t, e], e))
        ids[t, :len(order[:k])] = order[:k]
    return ids


def weights(logits, ids, renorm):
    T, k = ids.shape
    x = logits.astype(np.float64)
    w = np.zeros((T, k))
    for t in range(T):
        sel = ids[t][ids[t] >= 0]
        if sel.size == 0:
            continue
        e = np.exp(x[t, sel] - x[t, sel].max())
        w[t, :sel.size] = e / (e.sum() if renorm else np.exp(x[t] - x[t, sel].max()).sum())
    return w


def plan(ids, groups, per_row):
    """(offsets, rows, slots), stable; ids outside belong to no group, their rows come last."""
    flat = ids.reshape(-1)
    key = np.where((flat >= 0) & (flat < groups), flat, groups)
    order = np.argsort(key, kind="stable")
    offsets = np.array([(key < g).sum() for g in range(groups + 1)], np.int32)
    rows = (order // per_row).astype(np.int32)
    slots = np.empty_like(order)
    slots[order] = np.arange(order.size)
    slots = np.where(key < groups, slots, -1).astype(np.int32).reshape(ids.shape)
    return offsets, rows, slots


def sizes_to_offsets(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
