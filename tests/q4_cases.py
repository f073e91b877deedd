"""Plain implementations, in 64 bits, of the 4-bit cache's operators and of the check of drafted tokens, for the tests."""
from __future__ import annotations

import numpy as np


def round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


# ---- the cache ----
def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """fp32 [..., D] -> f16 scales [..., D/32], codes [..., D] (the exact choice: 64 bits separate x / d from every border)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    safe = np.where(bad[..., None], np.float32(0), b)
    top = np.take_along_axis(safe, np.abs(safe).argmax(-1)[..., None], -1)
    d = np.clip(top * np.float32(-0.125), -65504, 65504).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d == 0, 8.0, np.clip(np.floor(safe.astype(np.float64) / d.astype(np.float64) + 8.5), 0, 15))
    d = np.where(bad[..., None], np.float16(np.nan), d)[..., 0]
    return d, c.reshape(x.shape).astype(np.uint8)


def held(x: np.ndarray) -> np.ndarray:
    d, c = quantise(x)
    return ((c.reshape(*d.shape, 32).astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(x.shape)


def pack(codes: np.ndarray) -> np.ndarray:
    """codes [kv_heads, slots, D] -> bytes [kv_heads, slots/8, D/32, 8, 16]."""
    h, s, d = codes.shape
    c = codes.reshape(h, s // 8, 8, d // 32, 32)
    return np.ascontiguousarray((c[..., :16] | (c[..., 16:] << 4)).transpose(0, 1, 3, 2, 4))


def unpack(data: np.ndarray) -> np.ndarray:
    h, s8, blocks, _, _ = data.shape
    c = data.transpose(0, 1, 3, 2, 4)
    return np.concatenate([c & 15, c >> 4], -1).reshape(h, s8 * 8, blocks * 32)


def values(data: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Packed codes and scales [kv_heads, slots, D/32] -> float64 [kv_heads, slots, D]."""
    c = unpack(data)
    return ((c.reshape(*scales.shape, 32).astype(np.float64) - 8) * scales.astype(np.float64)[..., None]).reshape(c.shape)


# ---- attention ----
def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, adjacent: bool) -> np.ndarray:
    """x fp32 [tokens, heads, D], tables fp32 [tokens, pairs]; fp32, every operation rounded."""
    pairs = cos.shape[1]
    y = x.copy()
    c, s = cos[:, None], sin[:, None]
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, filled: int, scale: float) -> tuple[np.ndarray, np.ndarray]:
    """q [tokens, heads, D] (rotated), k and v [kv_heads, filled + tokens, D] as the cache holds them -> out [tokens, heads, D], weights
    [kv_heads, filled + tokens] summed over tokens and the group."""
    tokens, heads, d = q.shape
    group = heads // k.shape[0]
    out, received = np.empty((tokens, heads, d)), np.zeros(k.shape[:2])
    hidden = np.arange(filled + tokens)[None] > filled + np.arange(tokens)[:, None]
    for h in range(heads):
        kk, vv = k[h // group], v[h // group]
        with np.errstate(invalid="ignore"):
            s = np.where(hidden, -np.inf, (q[:, h].astype(np.float64) @ kk.T) * scale)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[:, h] = np.where(hidden[:, :, None], 0.0, p[:, :, None] * vv[None]).sum(1) if not np.isfinite(vv).all() else p @ vv
        received[h // group] += np.where(hidden, 0.0, p).sum(0)
    return out, received


# ---- eviction ----
def kept_slots(weight: np.ndarray, filled: int, keep: int, first: int, last: int) -> np.ndarray:
    """weight [kv_heads, slots] -> the kept slots [kv_heads, min(filled, keep)], ascending."""
    found = []
    for row in weight[:, :filled]:
        rank = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
        nan = np.isnan(row)
        if filled <= keep:
            found.append(np.arange(filled))
            continue
        middle = np.arange(first, filled - last)
        order = middle[np.lexsort((middle, nan[middle], -rank[middle]))]      # larger first, NaN behind -inf, then the lowest slot
        found.append(np.sort(np.concatenate([np.arange(first), order[:keep - first - last], np.arange(filled - last, filled)])))
    return np.array(found)


# ---- drafted tokens ----
def distribution(row: np.ndarray, temperature: float, top_k: int, top_p: float) -> np.ndarray | None:
    """p of one row of logits, in order of id; None without a finite logit."""
    ids = np.flatnonzero(np.isfinite(row))
    if not ids.size:
        return None
    if temperature == 0:
        temperature, top_k, top_p = 1.0, 1, 1.0
    x = row[ids].astype(np.float64)
    order = np.lexsort((ids, -x))
    if top_k:
        order = order[:top_k]
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp((x[order] - x[order[0]]) / float(np.float32(temperature)))
    e /= e.sum()
    if 0 < top_p < 1:
        n = min(int(np.searchsorted(np.cumsum(e), float(np.float32(top_p)))) + 1, e.size)
        order, e = order[:n], e[:n] / e[:n].sum()
    p = np.zeros(row.size)
    p[ids[order]] = e
    return p


def verify(logits, tokens, q, uniforms, temperature, top_k, top_p):
    """q [drafts, vocab] or None (certain drafts) -> out [drafts + 1], accepted, probs [drafts]."""
    drafts, vocab = len(tokens), logits.shape[1]
    p = [distribution(row, temperature, top_k, top_p) for row in logits]
    ok = [0 <= t < vocab and p[i] is not None for i, t in enumerate(tokens)]
    probs = np.array([p[i][t] if ok[i] else 0.0 for i, t in enumerate(tokens)])
    accepted = 0
    while accepted < drafts and ok[accepted] and uniforms[accepted] * (1.0 if q is None else q[accepted, tokens[accepted]]) < probs[accepted]:
        accepted += 1
    out = np.full(drafts + 1, -1, np.int64)
    out[:accepted] = tokens[:accepted]
    row = p[accepted]
    if row is not None:
        rest = row.copy()
        if accepted < drafts:
            if q is not None:
                rest = np.maximum(row - q[accepted], 0)
            elif 0 <= tokens[accepted] < vocab:
                rest[tokens[accepted]] = max(rest[tokens[accepted]] - 1.0, 0.0)
        if not rest.sum() > 0:
            rest = row
        cum = np.cumsum(rest)
        out[accepted] = np.flatnonzero((cum >= uniforms[drafts] * cum[-1]) & (rest > 0))[0]
    return out, accepted, probs
