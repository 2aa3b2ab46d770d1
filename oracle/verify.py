"""Oracle of the verification of drafted tokens, in fp64 on the CPU, token by token."""

from __future__ import annotations

import math


def _softmax(row, T):
    row = [float(z) for z in row]
    if any(math.isnan(z) or z == math.inf for z in row):
        return None
    m = max(row)
    if m == -math.inf:
        return None
    e = [math.exp((z - m) / T) for z in row]
    s = math.fsum(e)
    return [x / s for x in e]


def verify(logits, drafts, uniform, T, draft_logits=None, lengths=None, greedy=False):
    """(tokens, accepted, logp) as lists; logits [S, K + 1, V]."""
    tokens, accepted, logp = [], [], []
    S, rows, V = logits.shape
    K = rows - 1
    for s in range(S):
        n = K if lengths is None else min(max(int(lengths[s]), 0), K)
        out, lps = [], []
        left = None
        for i in range(n + 1):
            p = _softmax(logits[s, i].tolist(), T)
            left = p
            if i == n:
                break
            x = int(drafts[s, i])
            ok = False
            if greedy:
                ok = p is not None and x == max(range(V), key=lambda v: (float(logits[s, i, v]), -v))
            elif 0 <= x < V and p is not None:
                q = [1.0 if v == x else 0.0 for v in range(V)] if draft_logits is None else \
                    _softmax(draft_logits[s, i].tolist(), T)
                if q is not None:
                    ok = float(uniform[s, i]) * q[x] < p[x]
                    if not ok:
                        r = [max(a - b, 0.0) for a, b in zip(p, q)]
                        left = r if math.fsum(r) > 0 else p
            if not ok:
                break
            out.append(x)
            lps.append(math.log(p[x]))
        accepted.append(len(out))
        if p is None:
            out.append(-1)
            lps.append(math.nan)
        elif greedy:
            z = logits[s, len(out)]
            v = max(range(V), key=lambda v: (float(z[v]), -v))
            out.append(v)
            lps.append(math.log(p[v]))
        else:
            t = float(uniform[s, K]) * math.fsum(left)
            cum, got = 0.0, -1
            for v in range(V):
                if left[v] > 0:
                    got = v
                    if cum + left[v] > t:
                        break
                cum += left[v]
            out.append(got)
            lps.append(math.log(p[got]))
        tokens.append(out + [-1] * (rows - len(out)))
        logp.append(lps + [0.0] * (rows - len(lps)))
    return tokens, accepted, logp


def verify_dense(logits, drafts, uniform, T, draft_logits=None, lengths=None):
    """The same by whole rows of tensors, for large vocabularies; rows with a softmax only."""
    import torch
    S, rows, V = logits.shape
    K = rows - 1
    tokens = torch.full((S, rows), -1, dtype=torch.int64)
    logp = torch.zeros(S, rows, dtype=torch.float64)
    accepted = torch.zeros(S, dtype=torch.int64)
    for s in range(S):
        n = K if lengths is None else min(max(int(lengths[s]), 0), K)
        lp = torch.log_softmax(logits[s].double() / T, 1)
        lq = None if draft_logits is None else torch.log_softmax(draft_logits[s].double() / T, 1)
        a = 0
        while a < n:
            x = int(drafts[s, a])
            qx = 1.0 if lq is None else lq[a, x].exp().item()
            if not float(uniform[s, a]) * qx < lp[a, x].exp().item():
                break
            tokens[s, a], logp[s, a] = x, lp[a, x]
            a += 1
        r = lp[a].exp()
        if a < n:
            less = r.clone()
            if lq is None:
                less[int(drafts[s, a])] = 0.0
            else:
                less = (r - lq[a].exp()).clamp(min=0.0)
            r = less if less.any() else r
        cum = r.cumsum(0)
        v = int((cum <= float(uniform[s, K]) * cum[-1]).sum())
        v = min(v, int(r.nonzero()[-1, 0]))
        tokens[s, a], logp[s, a], accepted[s] = v, lp[a, v], a
    return tokens, accepted, logp
