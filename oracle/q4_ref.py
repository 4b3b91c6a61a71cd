"""Float64 references of the 4-bit operators and of token log probabilities, in numpy: from their
formulas, without the package."""
from __future__ import annotations

import numpy as np


def unpack(codes: np.ndarray) -> np.ndarray:
    """Codes 0..15 of packed bytes [..., n / 2], the even element in the low half."""
    out = np.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=np.float64)
    out[..., 0::2], out[..., 1::2] = codes & 15, codes >> 4
    return out


def w4_weight(qweight, scales, zeros=None) -> np.ndarray:
    """scale (u - zero) [N, K] of codes [N, K/2], scales [N, K/G] and zeros [N, K/G] (8 if None)."""
    u = unpack(qweight)
    g = u.shape[1] // scales.shape[1]
    z = 8.0 if zeros is None else np.repeat(zeros.astype(np.float64), g, axis=1)
    return np.repeat(scales.astype(np.float64), g, axis=1) * (u - z)


def round_bf16(x: np.ndarray) -> np.ndarray:
    """Nearest bf16 (ties to even) of float32 values, as float64."""
    b = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.nan, r).astype(np.float64)


def kv4_quantize(x: np.ndarray, group: int):
    """(codes u 0..15, scales) of x [..., n] in groups: s = bf16(max|x| / 7), u = 8 + clamp(round(x / s))."""
    y = x.reshape(x.shape[:-1] + (-1, group)).astype(np.float64)
    amax = np.abs(y).max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        s = np.where(np.isfinite(amax), round_bf16((amax / 7).astype(np.float32)), np.nan)
        q = np.where(s[..., None] > 0, np.round(y / s[..., None]), 0.0)
    return (np.clip(q, -7, 7) + 8).reshape(x.shape), s


def kv4_values(u: np.ndarray, s: np.ndarray) -> np.ndarray:
    g = u.shape[-1] // s.shape[-1]
    return np.repeat(s, g, axis=-1) * (u - 8.0)


def attend(q, k, v, lengths, scale):
    """q [B, T, Hq, D] over k, v [B, Hk, S, D]: query i of sequence b sees positions
    0 .. lengths[b] - T + i (below S); none: 0."""
    B, T, Hq, D = q.shape
    Hk, S = k.shape[1], k.shape[2]
    out = np.zeros(q.shape)
    for b in range(B):
        for t in range(T):
            n = min(int(lengths[b]) - T + t + 1, S)
            if n <= 0:
                continue
            for h in range(Hq):
                hk = h // (Hq // Hk)
                z = (k[b, hk, :n] @ q[b, t, h]) * scale
                p = np.exp(z - z.max())
                out[b, t, h] = (p @ v[b, hk, :n]) / p.sum()
    return out


def token_logprobs(x: np.ndarray, tokens, top_k: int):
    """(logprobs, entropy, top_logprobs, top_tokens) of rows x [R, V] (float64)."""
    R, V = x.shape
    lp, ent = np.empty(R), np.empty(R)
    top, at = np.empty((R, top_k)), np.empty((R, top_k), dtype=np.int64)
    for r in range(R):
        row, tok = x[r], int(tokens[r])
        order = np.arange(V) if np.isnan(row).any() else np.argsort(-row, kind="stable")
        at[r] = order[:top_k]
        m = row.max()
        if np.isnan(m) or m == np.inf:
            lp[r] = ent[r] = np.nan
            top[r] = np.nan
            continue
        if m == -np.inf:
            lp[r], ent[r], top[r] = -np.inf, 0.0, -np.inf
            continue
        e = np.exp(row - m)
        # x - m first: m + log s would lose log s next to an m of the type's lowest value
        d, p = row - m - np.log(e.sum()), e / e.sum()
        lp[r] = d[tok] if 0 <= tok < V else -np.inf
        ent[r] = -(p[p > 0] * d[p > 0]).sum()
        top[r] = d[at[r]]
    return lp, ent, top, at
