"""Plain 64-bit statements of the decode-step operators, on rows by position: no pool layout, no library code."""
from __future__ import annotations

import numpy as np


def q4_stands_for(rows):
    """What a 4-bit pool keeps of f32 rows [.., d]: per group of 32 an offset rounded down and a step rounded up to f16,
    codes 0..15.  The arithmetic of the rule is f32's."""
    x = np.asarray(rows, np.float32).reshape(*rows.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        fits = (np.abs(x) <= 65504).all(-1, keepdims=True)  # (a NaN fails too)
        lo = x.min(-1, keepdims=True)
        z = lo.astype(np.float16)
        z = np.where(z.astype(np.float32) > lo, np.nextafter(z, np.float16(-np.inf)), z)
        want = (x.max(-1, keepdims=True) - z.astype(np.float32)) / np.float32(15)
        s = want.astype(np.float16)
        s = np.where(s.astype(np.float32) < want, np.nextafter(s, np.float16(np.inf)), s)
        sf = s.astype(np.float32)
        c = np.where(sf > 0, np.clip(np.rint((x - z.astype(np.float32)) / np.where(sf > 0, sf, 1)), 0, 15), 0)
        out = z.astype(np.float64) + s.astype(np.float64) * c.astype(np.float64)
    return np.where(fits, out, np.nan).reshape(rows.shape), np.where(fits, s, 0).astype(np.float64)


def stands_for(rows, dtype: str):
    """What a pool of `dtype` keeps of f32 rows, in f64."""
    if dtype == "q4":
        return q4_stands_for(rows)[0]
    if dtype == "f32":
        return rows.astype(np.float64)
    import torch
    t = torch.from_numpy(np.ascontiguousarray(rows, np.float32))
    return t.to(torch.bfloat16 if dtype == "bf16" else torch.float16).double().numpy()


def window_attention(q, k, v, window: int, sinks: int):
    """q [heads, d]; k, v [positions, kv_heads, d] of one token's sequence, the token at the last of them."""
    n, kvh, d = k.shape
    j = np.arange(n)
    seen = (j < sinks) | (j > n - 1 - window) if window else np.full(n, True)
    qg = np.asarray(q, np.float64).reshape(kvh, -1, d)
    k, v = k[seen].astype(np.float64), v[seen].astype(np.float64)
    s = np.einsum("ghd,pgd->ghp", qg, k) / np.sqrt(d)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("ghp,pgd->ghd", p, v).reshape(-1, d)


def head_prelude(x, w, eps, cos, sin):
    """x [tokens, heads, d] f64; w [d] or None; cos, sin [tokens, rot / 2] or None."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is not None:
        h = cos.shape[-1]
        a, b, c, s = x[..., :h], x[..., h:2 * h], cos[:, None], sin[:, None]
        x = np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)
    return x
