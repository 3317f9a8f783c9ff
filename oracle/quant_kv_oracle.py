"""Oracle of the rotary append and of the 8-bit paged KV cache, in numpy float64.

Restates the definitions (include/plastic_kv.h: pi_rope_append and the pi_*_q8 entry points)
token by token, without this package's code. Pools are physical [P, H, S, D]; an 8-bit pool is
held as the float64 values of its e4m3 elements, NaN included, and a scale per (page, head).
"""

from __future__ import annotations

import math

import numpy as np

MIN_EXP = -118
E4M3_MAX = 448.0


def rope_rows(x: np.ndarray, positions, inv_freq, interleaved: bool = False,
              rope_scale: float = 1.0, weight=None, eps: float = 1e-5) -> np.ndarray:
    """QK-norm (with a weight) and rotation of x [T, H, D]."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    f = np.asarray(inv_freq, np.float64)
    n = f.shape[0]
    angle = np.asarray(positions, np.float64)[:, None] * f[None, :]
    c, s = np.cos(angle)[:, None] * rope_scale, np.sin(angle)[:, None] * rope_scale
    i = 2 * np.arange(n) if interleaved else np.arange(n)
    j = i + 1 if interleaved else i + n
    out = x.copy()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., j] * c + x[..., i] * s
    return out


def e4m3_round(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value, ties to even, saturating; NaN stays NaN."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 1.0)
    with np.errstate(divide="ignore"):
        step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    with np.errstate(invalid="ignore"):
        r = np.round(x / step) * step
    return np.clip(r, -E4M3_MAX, E4M3_MAX)


def block_exp(values: np.ndarray) -> int:
    """Smallest e >= MIN_EXP with amax <= 448 * 2^e over the finite values."""
    v = np.abs(values[np.isfinite(values)])
    top = float(v.max()) if v.size else 0.0
    if top == 0.0:
        return MIN_EXP
    m, x = math.frexp(top)  # top = m * 2^x, 448 = 0.875 * 2^9
    return max(MIN_EXP, x - 9 + (1 if m > 0.875 else 0))


def runs(slots, page_size: int):
    """(first token, page, offset, length) of every run of consecutive slots inside a page."""
    slots = [int(s) for s in slots]
    out, t = [], 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        page, off = divmod(slots[t], page_size)
        n = 1
        while t + n < len(slots) and off + n < page_size and slots[t + n] == slots[t] + n:
            n += 1
        out.append((t, page, off, n))
        t += n
    return out


def append_q8(rows: np.ndarray, slots, pool: np.ndarray, scale: np.ndarray) -> None:
    """rows [T, H, D] into the blocks of pool [P, H, S, D] / scale [P, H], in place."""
    P, H, S, _ = pool.shape
    for t, page, off, n in runs(slots, S):
        if page >= P:
            continue
        for h in range(H):
            new = rows[t:t + n, h]
            e = block_exp(new)
            if off:
                e = max(e, int(math.log2(scale[page, h])))
                if 2.0 ** e != scale[page, h]:
                    pool[page, h, :off] = e4m3_round(pool[page, h, :off] * (scale[page, h] / 2.0 ** e))
            scale[page, h] = 2.0 ** e
            pool[page, h, off:off + n] = e4m3_round(new / 2.0 ** e)


def attention_q8(q: np.ndarray, k_pool: np.ndarray, v_pool: np.ndarray, k_scale: np.ndarray,
                 v_scale: np.ndarray, tables, lens, scale: float | None = None) -> np.ndarray:
    """One query row [Hq, D] per entry of lens over its first lens[b] tokens: q [B, Hq, D],
    tables[b] the request's page ids. Rows with nothing to see are zero."""
    B, Hq, D = q.shape
    H, S = k_pool.shape[1], k_pool.shape[2]
    G = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = np.zeros((B, Hq, D))
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        ids = np.asarray(tables[b][:-(-n // S)], dtype=np.int64)
        k = (k_pool[ids] * k_scale[ids][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :n]
        v = (v_pool[ids] * v_scale[ids][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :n]
        for h in range(H):
            x = (q[b, h * G:(h + 1) * G].astype(np.float64) @ k[h].T) * scale
            x = np.exp(x - x.max(-1, keepdims=True))
            out[b, h * G:(h + 1) * G] = (x @ v[h]) / x.sum(-1, keepdims=True)
    return out
