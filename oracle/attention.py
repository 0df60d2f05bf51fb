"""Softmax attention and its gradients from their formulas in float64 (numpy).

Arrays are [batch, length, heads, dim]; key heads are shared by heads / kv_heads query heads. The
backward pass takes the forward's out and lse as given, as the kernels do."""
from __future__ import annotations

import numpy as np


def seen(b: int, n: int, m: int, causal: bool, key_mask) -> np.ndarray:
    """[b, 1, n, m] truth values: whether query i sees key j."""
    s = np.ones((b, 1, n, m), bool)
    if causal:
        s &= (np.arange(m)[None, :] <= np.arange(n)[:, None] + (m - n))[None, None]
    if key_mask is not None:
        s &= np.asarray(key_mask, bool)[:, None, None, :]
    return s


def heads_first(x, group: int = 1) -> np.ndarray:
    """[b, heads * group, n, d] in float64."""
    return np.repeat(np.asarray(x, np.float64).transpose(0, 2, 1, 3), group, axis=1)


def _visible(x, key_mask, group):
    """As heads_first, zeros in the rows of keys that the mask hides (what they hold does not matter)."""
    x = heads_first(x, group)
    return x if key_mask is None else np.where(np.asarray(key_mask, bool)[:, None, :, None], x, 0.0)


def forward(q, k, v, scale, causal=False, key_mask=None):
    """(out [b, n, h, d], lse [b, h, n], probabilities [b, h, n, m])"""
    g = q.shape[2] // k.shape[2]
    Q, K, V = heads_first(q), _visible(k, key_mask, g), _visible(v, key_mask, g)
    see = seen(q.shape[0], q.shape[1], k.shape[1], causal, key_mask)
    s = np.where(see, scale * (Q @ K.transpose(0, 1, 3, 2)), -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    base = np.where(np.isneginf(top), 0.0, top)
    e = np.exp(s - base)
    total = e.sum(-1, keepdims=True)
    p = np.divide(e, total, out=np.zeros_like(e), where=total != 0)
    with np.errstate(divide="ignore"):
        lse = (np.log(total) + base)[..., 0]
    return (p @ V).transpose(0, 2, 1, 3), lse, p


def backward(dout, q, k, v, out, lse, scale, causal=False, key_mask=None):
    """(dq, dk, dv, p, ds): gradients, and the probabilities and score gradients [b, h, n, m] they come from."""
    g = q.shape[2] // k.shape[2]
    Q, K, V, O, DO = heads_first(q), _visible(k, key_mask, g), _visible(v, key_mask, g), heads_first(out), heads_first(dout)
    see = seen(q.shape[0], q.shape[1], k.shape[1], causal, key_mask)
    row = np.asarray(lse, np.float64)[..., None]
    s = np.where(see, scale * (Q @ K.transpose(0, 1, 3, 2)), -np.inf)
    p = np.where(see, np.exp(s - np.where(np.isneginf(row), 0.0, row)), 0.0)
    ds = scale * p * (DO @ V.transpose(0, 1, 3, 2) - (DO * O).sum(-1, keepdims=True))
    dq = ds @ K

    def shared(x):  # sum over the query heads of a key head
        b, h, m, d = x.shape
        return x.reshape(b, h // g, g, m, d).sum(2).transpose(0, 2, 1, 3)

    return dq.transpose(0, 2, 1, 3), shared(ds.transpose(0, 1, 3, 2) @ Q), shared(p.transpose(0, 1, 3, 2) @ DO), p, ds
