"""Error bounds of the 4-bit operators and of token log probabilities, derived from the number
formats: u = 2^-24 is half a step of fp32 next to 1, and every output is rounded once more to its own
type (half a step, finfo.eps / 2 relative).

w4: a group's sum of G products and a bias of up to 32 times the row sum is held in fp32; its partial
sums are at most 48 sum|x| s (codes up to 15, offsets up to 31), with at most one rounding per four
products, and then K / G group sums are added.

attend: scores are fp32 sums of D products in the same form, so a score is off by about
u * 48 * sqrt(D / 4) * scale * sum|q| s_k, which the weights have as relative error; weights keep at
least 16 bits, and the value sums carry the same offset: for the tests' inputs (unit keys and
queries, D <= 128) below 2e-4 of the largest value.

log probabilities: e^d is within 2^-22 (the argument's rounding, |d| log2 e u, and the unit's own),
sums of V of them within 2^-20 relative, x - m - log s within 2 u |x| more: 1e-5 at |x| <= 40.
"""
import numpy as np
import torch

U = 2.0 ** -24
ATTEND_ABS = 2e-4
LOGPROB_ABS = 1e-5


def half_step(y: np.ndarray, dtype) -> np.ndarray:
    """Half a step of `dtype` at |y| (normal range; the smallest normal below it)."""
    info = torch.finfo(dtype)
    return info.eps / 2 * np.maximum(np.abs(y), info.tiny)


def w4_bound(x, w_scales, y, k, group, dtype):
    """|error| of y [M, N] for x [M, K] and scales [N, K / G] (float64 arrays)."""
    mass = np.abs(x).reshape(x.shape[0], -1, group).sum(-1) @ np.abs(w_scales).T      # [M, N]
    return half_step(y, dtype) * 1.01 + (group / 4 + k / group + 8) * U * 48 * mass
