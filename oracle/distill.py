"""Oracle of the teacher's lists and of the divergence from them, in fp64 on the CPU, row by row from the definition."""

from __future__ import annotations

import math

import torch


def topk(z, T, k):
    """(ids [n, k], logp [n, k]): by value descending (NaN first, -0 as 0), equal values by column ascending."""
    z = z.double()
    ids = []
    for row in z.tolist():
        order = sorted(range(len(row)), key=lambda j: (0 if math.isnan(row[j]) else 1,
                                                       0.0 if math.isnan(row[j]) else -row[j], j))
        ids.append(order[:k])
    ids = torch.tensor(ids, dtype=torch.int64).reshape(z.shape[0], k)
    return ids, torch.log_softmax(z / T, 1).gather(1, ids)


def weights(ids, teacher, V, normalise=True):
    """q [n, K] fp64, 0 for an empty slot."""
    teacher = teacher.double()
    q = torch.zeros_like(teacher)
    for r in range(ids.shape[0]):
        keep = [k for k in range(ids.shape[1]) if 0 <= int(ids[r, k]) < V and teacher[r, k] != -math.inf]
        if keep:
            t = teacher[r, keep]
            q[r, keep] = torch.softmax(t, 0) if normalise else torch.exp(t)
    return q


def divergence(s, ids, teacher, normalise=True):
    """(kl [n], dkl/ds [n, V]) of softmax(s) from the lists; s fp64 [n, V] (logits over T, transformed)."""
    n, V = s.shape
    q = weights(ids, teacher, V, normalise)
    kl = torch.zeros(n, dtype=torch.float64)
    grad = torch.zeros(n, V, dtype=torch.float64)
    for r in range(n):
        lp = torch.log_softmax(s[r], 0)
        Q = 0.0
        spread = torch.zeros(V, dtype=torch.float64)
        for k in range(ids.shape[1]):
            if q[r, k] > 0:
                kl[r] += q[r, k] * (torch.log(q[r, k]) - lp[ids[r, k]])
                spread[ids[r, k]] += q[r, k]
                Q += q[r, k]
        if Q > 0:
            grad[r] = Q * lp.exp() - spread
    return kl, grad
