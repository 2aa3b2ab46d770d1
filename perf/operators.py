"""The work around the two ends of a vocabulary matrix that a trainer of a student model asks of this package, as timed
and compared cases.

A case is one pass through one operator:

  topk     the teacher's list: the k largest logits of each row, their tokens and log-probabilities
  columns  the divergence of a student's logits from the teacher's lists, and the logits' gradient
  head     the same from hidden rows and the vocabulary weight, without the logits: loss and gradients in one call
  lookup   the rows of the weight for a stream of tokens, scaled
  update   the gradient of that lookup, over the whole vocabulary

n rows or tokens, hidden width d, vocabulary V, lists of K tokens. Student logits have a standard deviation of about
2.5, the teacher's differ from them by noise; a twentieth of the rows have a shorter list (the tail of it is -1) and a
fiftieth none at all. Tokens are Zipf(1.1) over a permuted vocabulary, one in a hundred of them -1 (packing).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.bfloat16}
CAP = 30.0  # the soft-cap: z' = 30 tanh(z / 30)


def _case(op, n, V, dtype, d=0, K=0, T=1.0, softcap=False, name=None):
    c = {"op": op, "n": n, "d": d, "V": V, "K": K, "dtype": dtype, "T": T, "softcap": softcap}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a served teacher answers for the one position it has just decoded: the smallest call
        _case("topk", 1, 151936, "bf16", K=64, name="topk-token"),
        # a 2,048-row chunk of a teacher's logits
        _case("topk", 2048, 151936, "bf16", K=64, name="topk-chunk"),
        # a small teacher checked in full precision, rows that start off a 16-byte boundary
        _case("topk", 333, 32003, "f32", K=20, name="topk-odd"),
        # the student's logits of the same chunk, produced by another module
        _case("columns", 2048, 151936, "bf16", K=64, name="columns-chunk"),
        # one short turn, an odd vocabulary, tempered
        _case("columns", 57, 128257, "f16", K=16, T=0.7, name="columns-turn"),
        # an ordinary micro-batch of the width and vocabulary the benchmark trains: the largest
        _case("head", 8192, 151936, "bf16", d=2560, K=64, name="head-batch"),
        # one short turn of a small model
        _case("head", 225, 32000, "bf16", d=1024, K=32, name="head-turn"),
        # a frozen fp8 head (adapters train): the gradient of the hidden rows alone
        _case("head", 4000, 151936, "fp8", d=2560, K=20, name="head-fp8"),
        # a decoding step of 16 sequences
        _case("lookup", 16, 128256, "bf16", d=4096, name="lookup-step"),
        # a packed prefix-tree micro-batch
        _case("lookup", 32768, 151936, "bf16", d=2560, name="lookup-packed"),
        # its gradient
        _case("update", 32768, 151936, "bf16", d=2560, name="update-packed"),
        # a short batch of a soft-capped model's width, in f16
        _case("update", 1501, 64000, "f16", d=2304, name="update-short"),
    ]


def draw(rng):
    def spread(lo, hi):  # even over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["topk", "columns", "head", "lookup", "update"])
    d, V = rng.choice([(1024, 32000), (2304, 64000), (2560, 151936), (4096, 128256)])
    V = max(1, V - rng.choice([0, 0, 1, 3, 64, 250]))
    K = rng.choice([1, 5, 16, 20, 32, 50, 64, 100, 128])
    T = rng.choice([1.0, 1.0, 0.7])
    if op == "topk":
        return _case(op, spread(1, 4096), V, rng.choice(["bf16", "bf16", "f16", "f32"]), K=K, T=T)
    if op == "columns":
        return _case(op, spread(8, 2048), V, rng.choice(["bf16", "bf16", "f16", "f32"]), K=K, T=T)
    if op == "head":
        n = spread(8, min(16384, 8192 * 2560 * 151936 // (d * V)))
        return _case(op, n, V, rng.choice(["bf16", "bf16", "f16", "fp8"]), d=d, K=K, T=T, softcap=rng.random() < 0.25)
    d -= rng.choice([0, 0, 8, 1])
    return _case(op, spread(1 if op == "lookup" else 8, 65536), V, rng.choice(["bf16", "bf16", "f16", "f32"]), d=d)


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tokens(g, n, V):
    p = 1.0 / torch.arange(1, V + 1, device="cuda", dtype=torch.float64) ** 1.1
    ranks = torch.multinomial(p.float(), n, replacement=True, generator=g)
    ids = torch.randperm(V, generator=g, device="cuda")[ranks]
    ids[torch.rand(n, generator=g, device="cuda") < 0.01] = -1
    return ids


def _shorten(g, ids):
    n, K = ids.shape
    u = torch.rand(n, generator=g, device="cuda")
    keep = torch.full((n,), K, device="cuda")
    keep[u < 0.07] = max(1, K // 2)
    keep[u < 0.02] = 0
    ids[torch.arange(K, device="cuda")[None, :] >= keep[:, None]] = -1


def prepare(case, seed):
    g = _gen(seed)
    op, n, d, V, K, T = (case[k] for k in ("op", "n", "d", "V", "K", "T"))
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    share = 1.0 if case["dtype"] == "f16" else 1.0 / n  # a row's part of the loss; f16 is trained with a loss scale
    if op in ("topk", "columns"):
        st["logits"] = (_normal(g, n, V) * 2.5).to(dt)
    if op == "columns":
        ids = torch.empty(n, K, dtype=torch.int64, device="cuda")
        teacher = torch.empty(n, K, device="cuda")
        for r in range(0, n, 256):
            z = st["logits"][r:r + 256].float()
            z = (z + _normal(g, *z.shape)) / T
            top = z.topk(K, dim=1)
            ids[r:r + 256] = top.indices
            teacher[r:r + 256] = top.values - z.logsumexp(1, keepdim=True)
        _shorten(g, ids)
        st.update(ids=ids, teacher=teacher, g=torch.rand(n, generator=g, device="cuda") * share)
        st["logits"].requires_grad_(True)
    if op == "head":
        rows = _normal(g, n, d).to(dt)
        w = _normal(g, V, d) * (2.5 / math.sqrt(d))
        scale = None
        if case["dtype"] == "fp8":
            scale = (w.abs().amax(1) / 448.0).clamp_min(1e-12)
            wt = (w / scale[:, None]).to(torch.float8_e4m3fn)
        else:
            wt = w.to(dt)
        ids = torch.empty(n, K, dtype=torch.int64, device="cuda")
        teacher = torch.empty(n, K, device="cuda")
        wb = w.to(torch.bfloat16)
        del w
        for r in range(0, n, 1024):  # the teacher's hidden rows differ from the student's by noise
            h = rows[r:r + 1024].float()
            h = (h + 0.3 * _normal(g, *h.shape)).to(torch.bfloat16)
            z = torch.matmul(h, wb.T).float()
            if case["softcap"]:
                z = CAP * torch.tanh(z / CAP)
            z = z / T
            top = z.topk(K, dim=1)
            ids[r:r + 1024] = top.indices
            teacher[r:r + 1024] = top.values - z.logsumexp(1, keepdim=True)
        del wb
        _shorten(g, ids)
        weight = (torch.rand(n, generator=g, device="cuda") < 0.9).float() * share
        st.update(rows=rows.requires_grad_(True), weight=wt.requires_grad_(scale is None), w_scale=scale, ids=ids,
                  teacher=teacher, row_weight=weight)
    if op in ("lookup", "update"):
        st["ids"] = _tokens(g, n, V)
        st["scale"] = math.sqrt(d)
    if op == "lookup":
        st["weight"] = (_normal(g, V, d) * 0.02).to(dt)
    if op == "update":
        st["grad"] = (_normal(g, n, d) * 0.01).to(dt)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state)


def _own(st):
    from octopus_amd import distill_op, embed_op
    from octopus_amd.head_op import Post

    case = st["case"]
    op, T = case["op"], case["T"]
    if op == "topk":
        ids, logp = distill_op.head_topk(st["logits"], T, case["K"])
        return {"ids": ids, "logp": logp}
    if op == "columns":
        kl = distill_op.distill_columns(st["logits"], T, st["ids"], st["teacher"])
        (grad,) = torch.autograd.grad(kl, st["logits"], st["g"])
        return {"kl": kl.detach(), "grad": grad}
    if op == "head":
        post = Post(1.0 / CAP, CAP, True) if case["softcap"] else Post()
        loss, kl = distill_op.fused_distill_head(st["rows"], st["weight"], st["ids"], st["teacher"], T,
                                                 st["row_weight"], post=post, w_scale=st["w_scale"])
        wrt = [t for t in (st["rows"], st["weight"]) if t.requires_grad]
        grads = torch.autograd.grad(loss, wrt)
        return {"loss": loss.detach(), "kl": kl, "grads": list(grads)}
    if op == "lookup":
        return embed_op.embed_rows(st["weight"], st["ids"], st["scale"])
    return embed_op.embed_bwd(st["grad"], st["ids"], case["V"], st["scale"])


def _plain_kl(logp, ids, teacher):
    """(kl [n], the teacher's probabilities [n, K], the ids with 0 for an empty slot)."""
    ok = (ids >= 0) & (ids < logp.shape[1])
    safe = torch.where(ok, ids, torch.zeros_like(ids))
    t = torch.where(ok, teacher, torch.full_like(teacher, -math.inf))
    m = t.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(t - m)
    s = e.sum(1, keepdim=True)
    none = s == 0
    q = e / torch.where(none, torch.ones_like(s), s)
    logq = t - m - torch.log(torch.where(none, torch.ones_like(s), s))
    term = q * (logq - logp.gather(1, safe))
    return torch.where(q > 0, term, torch.zeros_like(term)).sum(1), q, safe


def _plain(st):
    case = st["case"]
    op, T, V = case["op"], case["T"], case["V"]
    if op == "topk":
        z = st["logits"].float()
        top = torch.sort(z, dim=1, descending=True, stable=True)
        ids, z = top.indices[:, :case["K"]].contiguous(), z / T
        m = z.amax(1, keepdim=True)
        lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
        return {"ids": ids, "logp": z.gather(1, ids) - lse}
    if op == "columns":
        with torch.no_grad():
            s = st["logits"].float() / T
            m = s.amax(1, keepdim=True)
            logp = s - m - torch.log(torch.exp(s - m).sum(1, keepdim=True))
            kl, q, safe = _plain_kl(logp, st["ids"], st["teacher"])
            dz = torch.exp(logp) * q.sum(1, keepdim=True)
            dz.scatter_add_(1, safe, -q)
            return {"kl": kl, "grad": (dz * (st["g"][:, None] / T)).to(st["logits"].dtype)}
    if op == "head":
        with torch.no_grad():
            h = st["rows"].float()
            w = st["weight"].float()
            if st["w_scale"] is not None:
                w = w * st["w_scale"][:, None]
            z = torch.matmul(h, w.T)
            slope = None
            if case["softcap"]:
                z = torch.tanh(z / CAP)
                slope = 1 - z * z
                z = CAP * z
            s = z / T
            m = s.amax(1, keepdim=True)
            logp = s - m - torch.log(torch.exp(s - m).sum(1, keepdim=True))
            kl, q, safe = _plain_kl(logp, st["ids"], st["teacher"])
            dz = torch.exp(logp) * q.sum(1, keepdim=True)
            dz.scatter_add_(1, safe, -q)
            dz = dz * (st["row_weight"][:, None] / T)
            if slope is not None:
                dz = dz * slope
            grads = [torch.matmul(dz, w).to(st["rows"].dtype)]
            if st["w_scale"] is None:
                grads.append(torch.matmul(dz.T, h).to(st["weight"].dtype))
            return {"loss": (st["row_weight"] * kl).sum(), "kl": kl, "grads": grads}
    ok = (st["ids"] >= 0) & (st["ids"] < V)
    safe = torch.where(ok, st["ids"], torch.zeros_like(st["ids"]))
    with torch.no_grad():
        if op == "lookup":
            x = st["weight"][safe].float() * st["scale"]
            return torch.where(ok[:, None], x, torch.zeros_like(x)).to(st["weight"].dtype)
        x = st["grad"].float() * (ok[:, None].float() * st["scale"])
        gw = torch.zeros(V, case["d"], device=x.device).index_add_(0, safe, x)
        return gw.to(st["grad"].dtype)


def work(case):
    op, n, d, V, K = (case[k] for k in ("op", "n", "d", "V", "K"))
    e = 4 if case["dtype"] == "f32" else 2
    if op == "topk":
        return {"bytes": n * V * e + 12 * n * K, "flops": 4 * n * V}
    if op == "columns":  # the logits once, their gradient once
        return {"bytes": 2 * n * V * e + 12 * n * K + 8 * n, "flops": 8 * n * V}
    if op == "head":
        fp8 = case["dtype"] == "fp8"
        lists = 12 * n * K + 8 * n
        if fp8:
            return {"bytes": V * d + 4 * V + 2 * n * d * 2 + lists, "flops": 4 * n * d * V}
        return {"bytes": 2 * V * d * 2 + 2 * n * d * 2 + lists, "flops": 6 * n * d * V}
    if op == "lookup":  # at most n rows read, n written
        return {"bytes": 2 * n * d * e + 8 * n, "flops": n * d}
    return {"bytes": n * d * e + V * d * e + 8 * n, "flops": n * d}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _exact_list(row_logp, ids, teacher):
    """kl of one block of rows and minus its gradient in the log-probabilities, both dense."""
    V, K = row_logp.shape[1], ids.shape[1]
    hide = ~((ids >= 0) & (ids < V))
    q = torch.softmax(teacher.masked_fill(hide, -math.inf), 1).masked_fill(hide, 0.0)
    at = ids.clamp(0, V - 1)
    terms = torch.special.xlogy(q, q) - q * torch.gather(row_logp, 1, at)
    spread = torch.zeros_like(row_logp)
    for k in range(K):  # one slot at a time: no slot of a row is added twice at once
        col = at[:, k:k + 1]
        spread.scatter_(1, col, spread.gather(1, col) + q[:, k:k + 1])
    return terms.sum(1), spread, q.sum(1)


def exact(case, seed):
    st = prepare(case, seed)
    op, T, V, K = (case[k] for k in ("op", "T", "V", "K"))
    with torch.no_grad():
        if op == "topk":
            ids, logp = [], []
            for z in st["logits"].split(256):
                z = z.double()
                least = z.topk(K, dim=1).values[:, -1:]
                above, equal = z > least, z == least
                room = K - above.sum(1, keepdim=True)
                take = above | (equal & (equal.cumsum(1) <= room))
                cols = take.nonzero()[:, 1].reshape(-1, K)  # ascending
                order = torch.argsort(z.gather(1, cols), dim=1, descending=True, stable=True)
                cols = cols.gather(1, order)
                ids.append(cols)
                logp.append(torch.log_softmax(z / T, 1).gather(1, cols))
            return {"ids": torch.cat(ids), "logp": torch.cat(logp)}
        if op == "columns":
            kls, grads = [], []
            for r in range(0, case["n"], 256):
                lp = torch.log_softmax(st["logits"][r:r + 256].double() / T, 1)
                kl, spread, Q = _exact_list(lp, st["ids"][r:r + 256], st["teacher"][r:r + 256].double())
                kls.append(kl)
                grads.append((Q[:, None] * lp.exp() - spread) * st["g"][r:r + 256, None].double() / T)
            return {"kl": torch.cat(kls), "grad": torch.cat(grads)}
        if op == "head":
            w = st["weight"].float().double()
            if st["w_scale"] is not None:
                w *= st["w_scale"].double()[:, None]
            gw = torch.zeros_like(w) if st["w_scale"] is None else None
            kls, ghs = [], []
            for r in range(0, case["n"], 1024):
                h = st["rows"][r:r + 1024].double()
                z = h @ w.T
                cap = torch.tanh(z / CAP) if case["softcap"] else None
                lp = torch.log_softmax((z if cap is None else CAP * cap) / T, 1)
                kl, spread, Q = _exact_list(lp, st["ids"][r:r + 1024], st["teacher"][r:r + 1024].double())
                dz = (Q[:, None] * lp.exp() - spread) * (st["row_weight"][r:r + 1024, None].double() / T)
                if cap is not None:
                    dz *= 1 - cap ** 2
                kls.append(kl)
                ghs.append(dz @ w)
                if gw is not None:
                    gw += dz.T @ h
            kl = torch.cat(kls)
            return {"loss": st["row_weight"].double() @ kl, "kl": kl,
                    "grads": [torch.cat(ghs)] + ([gw] if gw is not None else [])}
        ids, s = st["ids"], st["scale"]
        used = (ids >= 0).nonzero()[:, 0]
        if op == "lookup":
            out = torch.zeros(case["n"], case["d"], dtype=torch.float64, device=ids.device)
            out[used] = st["weight"][ids[used]].double() * s
            return out
        gw = torch.zeros(V, case["d"], dtype=torch.float64, device=ids.device)
        return gw.index_put_((ids[used],), st["grad"][used].double() * s, accumulate=True)
