"""CPU oracle of the paged key/value cache and of sampling, in 64 bits -- test infrastructure only.

Restated from the formulas: per-head RMS norm (primitives.py:20-23), rotate-half
rotation (attention.py:66-70), GGUF Q4_0 blocks (gguf_dequant.py:25-46), causal
grouped-query attention (attention.py:59-115) with an optional window and sinks,
and the filters of the reference's ``sample`` (sampling.py:94-158) with the
random numbers as an input.
"""

from __future__ import annotations

import numpy as np


def norm_rotate(x, pos, cos_sin, w, eps):
    """x [T, H, D] float64 -> normalised (w not None) and rotated (cos_sin not None, rows = positions)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w.astype(np.float64)
    if cos_sin is None:
        return x
    d = x.shape[-1]
    c = cos_sin[pos].astype(np.float64)[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([a * c[..., 0] - b * c[..., 1], b * c[..., 0] + a * c[..., 1]], -1)


def q4_blocks(x):
    """fp32 rows [..., D] -> (codes uint8 [..., D], scales fp16 [..., D / 32])."""
    g = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    first = np.abs(g).argmax(-1)                              # the first of equals
    a = np.take_along_axis(g, first[..., None], -1)[..., 0]
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        d = (a / -8).astype(np.float16)
        q = np.floor(g / d.astype(np.float64)[..., None] + 8.5)
    q = np.where((d == 0)[..., None] | ~np.isfinite(d)[..., None] | bad[..., None], 8.0, np.clip(q, 0, 15))
    d = np.where(bad, np.float16(np.nan), d)
    return q.astype(np.uint8).reshape(x.shape), d


def q4_values(codes, d):
    g = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, 32) - 8
    with np.errstate(invalid="ignore"):
        return (g * d.astype(np.float64)[..., None]).reshape(codes.shape)


def nibble_dims(d, values):
    """The value that nibble j of a row of codes holds."""
    n, w = d // 32, 4 if values else 8
    return np.array([32 * ((j // w) % n) + w * ((j // w) // n) + j % w for j in range(d)])


class PoolView:
    """Rows of a pool given as numpy uint8 [pages, Hk, bytes]."""

    def __init__(self, pool, kv_type, d, page_size):
        self.p, self.kv, self.d, self.s = pool, kv_type, d, page_size

    def row(self, page, head, slot, values):
        """(codes in order of the values, scales) or the fp16 row."""
        half = self.p.shape[2] // 2
        b = self.p[page, head, half:] if values else self.p[page, head, :half]
        if self.kv == "F16":
            return b.view(np.float16).reshape(self.s, self.d)[slot]
        raw = b[:self.s * self.d // 2].reshape(self.s, self.d // 2)[slot]
        nib = np.stack([raw & 15, raw >> 4], -1).reshape(-1)
        codes = np.empty(self.d, np.uint8)
        codes[nibble_dims(self.d, values)] = nib
        return codes, b[self.s * self.d // 2:].view(np.float16).reshape(self.s, self.d // 32)[slot]

    def value(self, page, head, slot, values):
        r = self.row(page, head, slot, values)
        return r.astype(np.float64) if self.kv == "F16" else q4_values(*r)

    def keys_values(self, table, n, head):
        """float64 [n, D] keys and values of the first n positions of a sequence with pages `table`."""
        out = []
        for values in (False, True):
            rows = [self.value(int(table[p // self.s]), head, p % self.s, values) for p in range(n)]
            out.append(np.stack(rows) if rows else np.zeros((0, self.d)))
        return out


def visible(pos, n, window, sinks):
    """Which of the positions 0 .. n - 1 a row at position pos sees."""
    k = np.arange(n)
    ok = k <= pos
    if window > 0:
        ok &= (k > pos - window) | (k < sinks)
    return ok


def attention_row(q, k, v, seen, scale):
    """(output, sum p |v| / sum p, largest sum |q||k| scale, sum |v|) of one query row, float64."""
    if not seen.any():
        return np.zeros(v.shape[-1]), np.zeros(v.shape[-1]), 0.0, 0.0
    k, v = k[seen], v[seen]
    s = k @ q.astype(np.float64) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return (p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q.astype(np.float64))).max() * abs(scale)),
            np.abs(v).sum(0))


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share of the kept mass) of one row of logits."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return 0, -np.inf
    if not temperature > 0:
        return int(np.argmax(x)), 0.0
    if np.isposinf(x.max()):
        w = np.isposinf(x).astype(np.float64)
    else:
        w = np.where(np.isneginf(x), 0.0, np.exp((x - x.max()) / np.float64(temperature)))
    order = np.argsort(-x, kind="stable")
    n = min(top_k, len(x)) if top_k > 0 else len(x)
    p = w[order[:n]]
    before = np.cumsum(p) - p
    if top_p < 1:
        n = max(1, int((before < top_p * p.sum()).sum()))
    n = max(1, min(n, int((w[order[:n]] >= min(min_p, 1.0)).sum())))
    keep = np.zeros(len(x), bool)
    keep[order[:n]] = True
    m = np.where(keep, w, 0.0)
    c = np.cumsum(m)
    hit = np.flatnonzero(c > u * c[-1])
    i = int(hit[0]) if len(hit) else int(np.flatnonzero(m)[-1])
    return i, float(np.log(m[i] / c[-1]))
