"""Oracle of the embedding lookup and its gradient, in fp64 on the CPU, token by token."""

from __future__ import annotations

import torch


def lookup(w, ids, scale):
    out = torch.zeros(*ids.shape, w.shape[1], dtype=torch.float64)
    flat = out.reshape(-1, w.shape[1])
    for t, v in enumerate(ids.reshape(-1).tolist()):
        if 0 <= v < w.shape[0]:
            flat[t] = w[v].double() * scale
    return out


def gradient(grad, ids, V, scale, padding_idx=None):
    """(the gradient [V, d], the sums of the tokens' magnitudes [V, d], the tokens of each entry [V])."""
    d = grad.shape[-1]
    gw, mag, cnt = (torch.zeros(V, d, dtype=torch.float64), torch.zeros(V, d, dtype=torch.float64),
                    torch.zeros(V, dtype=torch.int64))
    g = grad.reshape(-1, d).double()
    for t, v in enumerate(ids.reshape(-1).tolist()):
        if 0 <= v < V and v != padding_idx:
            gw[v] += g[t] * scale
            mag[v] += g[t].abs() * abs(scale)
            cnt[v] += 1
    return gw, mag, cnt
