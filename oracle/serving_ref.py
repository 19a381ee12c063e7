"""CPU float64 oracle of the serving operators: per-head norm with rotation
(and its backward), paged attention of one new token, and sampling.

TEST INFRASTRUCTURE ONLY, like attention_ref: nothing in enilnets_b200/ uses it.
The rotation is nn/forward.py:80-88, the sampling order
generative/text_generation.py:118-134; the rest has no reference counterpart
and is written from the formulas.
"""
from __future__ import annotations

import itertools

import numpy as np


def norm_rope(x, w, eps, cos, sin):
    """x (..., S, H, D); cos, sin broadcastable to (..., S, 1, D / 2) or None."""
    x = np.asarray(x, np.float64)
    z = x if w is None else w * x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    if cos is None:
        return z
    h = x.shape[-1] // 2
    z1, z2 = z[..., :h], z[..., h:]
    return np.concatenate([z1 * cos - z2 * sin, z2 * cos + z1 * sin], -1)


def norm_rope_backward(dy, x, w, eps, cos, sin):
    """(dx, dw) for the gradient dy of norm_rope's output."""
    dy = np.asarray(dy, np.float64)
    h = dy.shape[-1] // 2
    dz = dy
    if cos is not None:
        d1, d2 = dy[..., :h], dy[..., h:]
        dz = np.concatenate([d1 * cos + d2 * sin, d2 * cos - d1 * sin], -1)
    if w is None:
        return dz, None
    x = np.asarray(x, np.float64)
    r = 1.0 / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    xh = x * r
    g = dz * w
    dx = r * (g - xh * np.mean(g * xh, -1, keepdims=True))
    return dx, (dz * xh).reshape(-1, dy.shape[-1]).sum(0)


def gather_pages(pages, table_row, positions):
    """(n, Hkv, D) rows of a (num_pages, Hkv, page_size, D) pool."""
    size = pages.shape[2]
    return np.stack([pages[table_row[j // size], :, j % size] for j in positions]) \
        if len(positions) else np.zeros((0, pages.shape[1], pages.shape[3]))


def visible(length, window, sinks):
    """Positions the query at length - 1 sees."""
    last = length - 1
    return [j for j in range(length)
            if window is None or last - j <= window or j < sinks]


def paged_decode(q, k_pages, v_pages, table, lens, *, window=None, sinks=0, slopes=None,
                 scale=None):
    """(out (B, H, D), lse (B, H)) in float64; an empty sequence: 0 and -inf."""
    B, H, D = q.shape
    Hkv = k_pages.shape[1]
    G = H // Hkv
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out, lse = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    for b in range(B):
        pos = visible(int(lens[b]), window, sinks)
        if not pos:
            continue
        K, V = gather_pages(k_pages, table[b], pos), gather_pages(v_pages, table[b], pos)
        dist = int(lens[b]) - 1 - np.asarray(pos, np.float64)
        for h in range(H):
            s = K[:, h // G] @ q[b, h] * scale
            if slopes is not None:
                s = s - slopes[h] * dist
            m = s.max()
            e = np.exp(s - m)
            out[b, h] = e @ V[:, h // G] / e.sum()
            lse[b, h] = m + np.log(e.sum())
    return out, lse


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row by the definition, in float64."""
    x = np.where(np.isnan(row), -np.inf, np.asarray(row, np.float64))
    top = x.max()
    if top == -np.inf:
        return -1
    order = np.argsort(-x, kind="stable")
    if temperature <= 0:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    ws = w[order].copy()
    if top_k > 0:
        ws[top_k:] = 0.0
    if top_p < 1.0:
        before = np.cumsum(ws) - ws
        drop = before >= top_p * ws.sum()
        drop[0] = False
        ws = np.where(drop, 0.0, ws)
    ws[ws < min(min_p, 1.0)] = 0.0
    kept = np.zeros_like(w)
    kept[order] = ws
    run = np.cumsum(kept)
    return int(np.searchsorted(run, u * run[-1], side="right"))


def sample_answers(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, eps=1e-5):
    """Tokens a computation with relative weight errors below eps may return:
    the draw and the thresholds each moved by eps either way."""
    if temperature <= 0:
        return {sample(row, u, temperature)}
    us = (max(0.0, u - eps), u, min(1.0 - 1e-12, u + eps))
    ps = (top_p,) if top_p >= 1.0 else (max(0.0, top_p - eps), top_p, top_p + eps)
    ms = (min_p,) if min_p <= 0.0 else (min_p * (1 - eps), min_p, min_p * (1 + eps))
    return {sample(row, a, temperature, top_k, b, c) for a, b, c in itertools.product(us, ps, ms)}
