"""Oracle of rows held in 8 bits and of the head's logits from them, in exact or 64-bit arithmetic on the CPU."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import torch

LEAST = 2.0 ** -119


def _round_even(x: Fraction) -> int:
    return round(x)  # Python rounds a Fraction's ties to even


def quantise(x, group=0, exact=False):
    """(q [n, d] int64, scale [n, groups] float64 holding fp32 values); exact: the quotients as fractions (slow)."""
    x = x.double().numpy() if isinstance(x, torch.Tensor) else np.asarray(x, dtype=np.float64)
    n, d = x.shape
    width = group or d
    groups = -(-d // width)
    q = np.zeros((n, d), dtype=np.int64)
    scale = np.zeros((n, groups))
    for j in range(groups):
        part = x[:, j * width:(j + 1) * width]
        a = np.abs(part).max(1)
        with np.errstate(invalid="ignore"):
            s = (a.astype(np.float32) * (np.float32(1) / np.float32(127))).astype(np.float64)
        s[a < LEAST] = 0.0
        s[~np.isfinite(a)] = np.nan
        scale[:, j] = s
        for r in range(n):
            if not s[r] > 0:
                continue
            if exact:
                q[r, j * width:j * width + part.shape[1]] = [_round_even(Fraction(float(v)) / Fraction(float(s[r])))
                                                            for v in part[r]]
            else:
                q[r, j * width:j * width + part.shape[1]] = np.rint(part[r] / s[r])
    return torch.from_numpy(q), torch.from_numpy(scale)


def widen(q, scale, group=0):
    d = q.shape[1]
    return q.double() * scale.double().repeat_interleave(group or d, 1)[:, :d]


def logits(x, wq, w_scale):
    """[n, V] in fp64 of rows x quantised a row each."""
    q, s = quantise(x)
    return (q.double() @ wq.double().T) * s * w_scale.double()


def grads(g, x, wq, w_scale):
    """(grad_rows, grad_w, and the sums of their terms' magnitudes) for g [n, V]."""
    q, s = quantise(x)
    xs, w = q.double() * s, wq.double() * w_scale.double()[:, None]
    g = g.double()
    return g @ w, g.T @ xs, g.abs() @ w.abs(), g.abs().T @ xs.abs()
