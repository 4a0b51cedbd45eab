"""Float64 oracle of the local attention and its learned position bias: the
definitions written out densely, one (batch, head) at a time, in numpy."""

from __future__ import annotations

import numpy as np


def bias_matrix(weight, table, n_q, n_k, q_start):
    """weight (H, nb), table (2 D + 1) -> (H, n_q, n_k), and the buckets (n_q, n_k)."""
    table = np.asarray(table)
    D = len(table) // 2
    delta = np.arange(n_q)[:, None] + q_start - np.arange(n_k)[None, :]
    buckets = table[np.clip(delta, -D, D) + D]
    return np.asarray(weight, dtype=np.float64)[:, buckets], buckets


def bias_grad(d_bias, buckets, nb):
    d_bias = np.asarray(d_bias, dtype=np.float64)
    return np.stack([np.bincount(buckets.ravel(), x.ravel(), nb) for x in d_bias]) if d_bias.shape[0] else \
        np.zeros((0, nb))


def visible_keys(n_q, n_k, q_start, causal, window, sinks, mask=None):
    """(n_q, n_k) bool; window None: all keys are near; mask (n_k,) or None."""
    j = np.arange(n_k)[None, :]
    delta = np.arange(n_q)[:, None] + q_start - j
    ok = np.ones_like(delta, dtype=bool)
    if window is not None:
        ok = (np.abs(delta) < window) | (j < sinks)
    if causal:
        ok &= delta >= 0
    if mask is not None:
        ok &= np.asarray(mask, dtype=bool)[None, :]
    return ok


def window_attn(q, k, v, *, causal=True, window=None, sinks=0, q_start=None, scale=None, weight=None, table=None,
                mask=None, d_o=None):
    """q (B,H,n_q,d), k, v (B,H_kv,n_k,d), mask (B,n_k).  Returns o, and with d_o
    also (d_q, d_k, d_v, d_weight or None)."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    B, H, n_q, d = q.shape
    H_kv, n_k = k.shape[1:3]
    G = H // H_kv
    q_start = n_k - n_q if q_start is None else q_start
    scale = d ** -0.5 if scale is None else scale
    bias, buckets = (None, None) if weight is None else bias_matrix(weight, table, n_q, n_k, q_start)
    o = np.zeros_like(q)
    if d_o is not None:
        d_o = np.asarray(d_o, dtype=np.float64)
        d_q, d_k, d_v = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
        d_w = None if weight is None else np.zeros(np.shape(weight))
    for b in range(B):
        ok = visible_keys(n_q, n_k, q_start, causal, window, sinks, None if mask is None else mask[b])
        seen = ok.any(0)  # a key that nobody sees takes no part, whatever it holds
        for h in range(H):
            K, V = (np.where(seen[:, None], x[b, h // G], 0.0) for x in (k, v))
            s = q[b, h] @ K.T * scale
            if bias is not None:
                s = s + bias[h]
            s = np.where(ok, s, -np.inf)
            top = s.max(1, keepdims=True, initial=-np.inf)
            e = np.exp(s - np.where(np.isfinite(top), top, 0.0))
            total = e.sum(1, keepdims=True)
            p = e / np.where(total > 0, total, 1.0)
            o[b, h] = p @ V
            if d_o is None:
                continue
            d_v[b, h // G] += p.T @ d_o[b, h]
            d_p = d_o[b, h] @ V.T
            d_s = p * (d_p - (p * d_p).sum(1, keepdims=True))
            d_q[b, h] = d_s @ K * scale
            d_k[b, h // G] += d_s.T @ q[b, h] * scale
            if d_w is not None:
                d_w[h] += np.bincount(buckets.ravel(), d_s.ravel(), d_w.shape[1])
    return o if d_o is None else (o, d_q, d_k, d_v, d_w)
