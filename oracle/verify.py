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
