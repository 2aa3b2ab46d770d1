"""The work around an 8-bit vocabulary matrix that a trainer and its rollouts ask of this package, as timed and compared
cases.

A case is one pass through one operator:

  logits  the head's logits from 8-bit integers: hidden rows quantised a row each, times weights quantised before
  train   the same with its gradients in the hidden rows and, straight through the rounding, in the weight
  held    activations held in 8 bits between a forward and its backward: written, and read back
  verify  drafted tokens checked against the target's probabilities: what is answered, and its log-probabilities

n rows, hidden width d, vocabulary V; S sequences of up to K drafts. Hidden rows have RMS 1 and a few wide columns, the
weights give logits with a standard deviation of about 2.5. Draft logits differ from the target's by noise, drafts are
sampled from them, one sequence in five drafts fewer than K tokens, and one in eight is held to 64 tokens by a mask.

What is quantised: over a row, or over each group of a row's values, with a the largest magnitude: scale = a / 127 in 32
bits, q = the quotient x / scale rounded to the nearest integer, ties to even (zeros where a < 2^-119).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LEAST = 2.0 ** -119


def _case(op, dtype, name=None, **sizes):
    c = dict({"op": op, "dtype": dtype, "n": 0, "d": 0, "V": 0, "S": 0, "K": 0, "T": 1.0, "group": 0, "draft": True,
              "greedy": False}, **sizes)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a served model decodes one sequence: the weight read once
        _case("logits", "bf16", "logits-token", n=1, d=2560, V=151936),
        # 64 sequences, four drafts each, verified in one pass
        _case("logits", "bf16", "logits-drafts", n=320, d=4096, V=128256),
        # a teacher's logits of a long prompt: the largest product
        _case("logits", "bf16", "logits-prompt", n=8192, d=2560, V=151936),
        # a small model of odd width and vocabulary in f16
        _case("logits", "f16", "logits-odd", n=333, d=1027, V=32003),
        # a chunk of a student that is trained for the 8-bit head it will be served with
        _case("train", "bf16", "train-chunk", n=2048, d=2560, V=151936),
        # one short turn of a small student in f16
        _case("train", "f16", "train-turn", n=225, d=1024, V=32000),
        # a layer's input over a packed prefix-tree micro-batch, held for its backward
        _case("held", "bf16", "held-packed", n=32768, d=2560, group=128),
        # a short batch of an odd width, a scale a row
        _case("held", "f16", "held-odd", n=1501, d=2303),
        # one sequence with four drafts: the smallest call
        _case("verify", "bf16", "verify-one", S=1, K=4, V=151936),
        # a decoding step of 64 sequences, tempered
        _case("verify", "bf16", "verify-step", S=64, K=4, V=128256, T=0.7),
        # drafts looked up in the prompt (no draft distribution), an odd vocabulary in full precision
        _case("verify", "f32", "verify-lookup", S=57, K=3, V=32003, draft=False),
        # a full rollout batch with long drafts
        _case("verify", "bf16", "verify-wide", S=256, K=7, V=151936),
    ]


def draw(rng):
    def spread(lo, hi):  # even over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logits", "logits", "train", "held", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d, V = rng.choice([(1024, 32000), (2304, 64000), (2560, 151936), (4096, 128256)])
    V = max(1, V - rng.choice([0, 0, 1, 3, 64, 250]))
    if op == "held":
        d -= rng.choice([0, 0, 8, 1])
        return _case(op, dtype, n=spread(8, 16384 if dtype == "f32" else 20480), d=d,
                     group=rng.choice([0, 0, 32, 64, 128, 256]))
    if op == "verify":
        K = rng.choice([0, 1, 2, 3, 4, 5, 7])
        most = 256 * 15 * 151936 * 2 // ((2 * K + 1) * V * (4 if dtype == "f32" else 2))
        return _case(op, dtype, S=spread(1, min(512, most)), K=K, V=V, T=rng.choice([1.0, 1.0, 0.7, 1.3]),
                     draft=rng.random() < 0.75, greedy=rng.random() < 0.2)
    d -= rng.choice([0, 0, 0, 8, 1])
    if op == "logits":
        return _case(op, dtype, n=spread(1, min(8192, 8192 * 2560 * 151936 // (d * V * (2 if dtype == "f32" else 1)))),
                     d=d, V=V)
    return _case(op, dtype, n=spread(8, 512 if dtype == "f32" else 2048), d=d, V=V)


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 6151 + 29)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, n, d):
    wide = torch.ones(d, device="cuda")
    wide[torch.randint(0, d, (max(1, d // 200),), generator=g, device="cuda")] = 6.0
    x = _normal(g, n, d) * wide
    return x / x.square().mean(1, keepdim=True).sqrt()


def _whole(x, scale):
    """x / scale to the nearest integer, in 64 bits."""
    safe = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    return torch.where(scale > 0, torch.round(x.double() / safe), torch.zeros_like(safe))


def _quantised(x, group=0):
    """(q as float, scale) of the rows of x [n, d]."""
    n, d = x.shape
    x = x.float()
    if not group:
        a = x.abs().amax(1)
        scale = torch.where(a < LEAST, torch.zeros_like(a), a / 127.0)
        return torch.cat([_whole(p, s[:, None]).float() for p, s in zip(x.split(8192), scale.split(8192))]), scale
    groups = -(-d // group)
    padded = torch.zeros(n, groups * group, device=x.device)
    padded[:, :d] = x
    q, scale = _quantised(padded.view(n * groups, group))
    return q.view(n, groups * group)[:, :d], scale.view(n, groups)


def _spread_scale(scale, d, group):
    return scale[:, None] if not group else scale.repeat_interleave(group, 1)[:, :d]


def prepare(case, seed):
    g = _gen(seed)
    op, n, d, V, S, K, T = (case[k] for k in ("op", "n", "d", "V", "S", "K", "T"))
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if op in ("logits", "train"):
        w = _normal(g, V, d) * (2.5 / math.sqrt(d))
        st["rows"] = _activations(g, n, d).to(dt).requires_grad_(op == "train")
        master = w.to(dt)
        del w
        # rows of 8-bit integers start on 16-byte boundaries, the bytes between them are zeros
        wq = torch.zeros(V, -(-d // 16) * 16, dtype=torch.int8, device="cuda")
        w_scale = torch.empty(V, device="cuda")
        for r in range(0, V, 16384):
            q, w_scale[r:r + 16384] = _quantised(master[r:r + 16384])
            wq[r:r + 16384, :d] = q.to(torch.int8)
        st.update(wq=wq[:, :d], w_scale=w_scale)
    if op == "train":
        st["weight"] = master.requires_grad_(True)
        grad = torch.softmax(_normal(g, n, V) * 2.5, 1)
        at = torch.randint(0, V, (n, 1), generator=g, device="cuda")
        grad.scatter_add_(1, at, torch.full((n, 1), -1.0, device="cuda"))
        grad *= _normal(g, n, 1) * (1.0 if case["dtype"] == "f16" else 1.0 / n)  # f16 is trained with a loss scale
        st["grad"] = grad.to(dt)
    if op == "held":
        st["x"] = _activations(g, n, d).to(dt)
    if op == "verify":
        z = _normal(g, S, K + 1, V) * 2.5
        only = (torch.arange(S, device="cuda") % 8 == 5).nonzero()[:, 0]
        keep = torch.randint(0, V, (S, 1, 64), generator=g, device="cuda")
        mask = torch.zeros(only.numel(), 1, V, dtype=torch.bool, device="cuda").scatter_(2, keep[only], True)
        draft = z[:, :K] + 0.7 * _normal(g, S, K, V)
        z[only] = z[only].masked_fill(~mask, -math.inf)
        draft[only] = draft[only].masked_fill(~mask, -math.inf)
        st["logits"], draft = z.to(dt), draft.to(dt)
        del z
        e = torch.empty(S, K, V, device="cuda").exponential_(generator=g)
        st["drafts"] = (draft.float() / T - torch.log(e)).argmax(2) if K else \
            torch.empty(S, 0, dtype=torch.int64, device="cuda")
        del e
        u = torch.rand(S, generator=g, device="cuda")
        st["lengths"] = torch.where(u < 0.2, (u * 5 * (K + 1)).long(), torch.full_like(u, K).long()).clamp_(0, K)
        st["uniform"] = torch.rand(S, K + 1, generator=g, device="cuda")
        st["draft_logits"] = draft if case["draft"] and not case["greedy"] else None
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state)


def _own(st):
    from octopus_amd import int8_op, verify_op

    case = st["case"]
    op = case["op"]
    if op == "logits":
        return int8_op.int8_head(st["rows"], st["wq"], st["w_scale"])
    if op == "train":
        z = int8_op.int8_head(st["rows"], st["wq"], st["w_scale"], weight=st["weight"])
        grads = torch.autograd.grad(z, (st["rows"], st["weight"]), st["grad"])
        return {"logits": z.detach(), "grads": list(grads)}
    if op == "held":
        q, scale = int8_op.quantise_rows(st["x"], case["group"])
        return {"scale": scale, "x": int8_op.widen_rows(q, scale, st["x"].dtype, case["group"])}
    tokens, accepted, logp = verify_op.verify_drafts(st["logits"], st["drafts"], st["uniform"], case["T"],
                                                     draft_logits=st["draft_logits"], lengths=st["lengths"],
                                                     greedy=case["greedy"])
    return {"tokens": tokens, "accepted": accepted, "logp": logp}


def _softmax(z, T):
    """(probabilities, log-probabilities) in 64 bits."""
    s = z.double() / T
    s = s - s.amax(-1, keepdim=True)
    e = torch.exp(s)
    total = e.sum(-1, keepdim=True)
    return e / total, s - torch.log(total)


def _plain(st):
    case = st["case"]
    op = case["op"]
    with torch.no_grad():
        if op in ("logits", "train"):
            dt = st["rows"].dtype
            qx, sx = _quantised(st["rows"])
            qw = st["wq"].float()
            z = (torch.matmul(qx, qw.T) * sx[:, None] * st["w_scale"]).to(dt)
            if op == "logits":
                return z
            g = st["grad"].float()
            dx = torch.matmul(g, qw * st["w_scale"][:, None]).to(dt)
            dw = torch.matmul(g.T, qx * sx[:, None]).to(dt)
            return {"logits": z, "grads": [dx, dw]}
        if op == "held":
            q, scale = _quantised(st["x"], case["group"])
            return {"scale": scale, "x": (q * _spread_scale(scale, case["d"], case["group"])).to(st["x"].dtype)}
        return _plain_verify(st, case)


def _plain_verify(st, case):
    S, K, T = case["S"], case["K"], case["T"]
    x, u, lengths = st["drafts"], st["uniform"].double(), st["lengths"]
    p, logp = _softmax(st["logits"], T)
    which = torch.arange(K + 1, device=x.device)
    if case["greedy"]:
        top = st["logits"].float().amax(2, keepdim=True)
        first = (st["logits"].float() == top).long().argmax(2)
        accept = x == first[:, :K]
    else:
        px = p[:, :K].gather(2, x[:, :, None])[:, :, 0]
        qx = torch.ones_like(px)
        if st["draft_logits"] is not None:
            q = _softmax(st["draft_logits"], T)[0]
            qx = q.gather(2, x[:, :, None])[:, :, 0]
        accept = u[:, :K] * qx < px
    accept = accept & (which[None, :K] < lengths[:, None])
    a = accept.long().cumprod(1).sum(1)
    at = torch.arange(S, device=x.device)
    if case["greedy"]:
        token = first[at, a]
    else:
        r = p[at, a]
        if K:
            rejected = (a < lengths)[:, None]
            k = a.clamp(max=K - 1)
            if st["draft_logits"] is not None:
                less = (r - q[at, k]).clamp(min=0)
            else:
                less = r.scatter(1, x[at, k][:, None], 0.0)
            rejected = rejected & (less.sum(1, keepdim=True) > 0)
            r = torch.where(rejected, less, r)
        cum = r.cumsum(1)
        token = (cum <= u[:, K:] * cum[:, -1:]).sum(1)
        last = r.shape[1] - 1 - (r > 0).flip(1).long().argmax(1)
        token = torch.minimum(token, last)
    tokens = torch.full((S, K + 1), -1, dtype=torch.int64, device=x.device)
    tokens[:, :K] = torch.where(which[None, :K] < a[:, None], x, tokens[:, :K])
    tokens[at, a] = token
    said = logp.gather(2, tokens.clamp(min=0)[:, :, None])[:, :, 0]
    return {"tokens": tokens, "accepted": a, "logp": torch.where(tokens >= 0, said, torch.zeros_like(said)).float()}


def work(case):
    op, n, d, V, S, K = (case[k] for k in ("op", "n", "d", "V", "S", "K"))
    e = 4 if case["dtype"] == "f32" else 2
    if op == "logits":
        return {"bytes": V * d + 4 * V + n * d * e + n * V * e, "flops": 2 * n * d * V}
    if op == "train":  # the logits as above, their gradient read, two gradients written
        return {"bytes": V * d + 4 * V + 2 * n * d * e + 2 * n * V * e + V * d * e, "flops": 6 * n * d * V}
    if op == "held":  # the values and what they are held as, each written and read
        scales = n * (-(-d // case["group"]) if case["group"] else 1)
        return {"bytes": 2 * n * d * e + 2 * (n * d + 4 * scales), "flops": 3 * n * d}
    rows = S * (2 * K + 1 if case["draft"] and not case["greedy"] else K + 1)
    return {"bytes": rows * V * e + 24 * S * (K + 1), "flops": 4 * rows * V}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _exact_rows(x):
    """The values that rows of x [n, d] stand for once held in 8 bits, and their scales."""
    x = x.double()
    a = x.abs().max(1).values
    scale = (a.float() / 127).double() * (a >= LEAST)
    steps = x / scale[:, None].clamp(min=1e-60)
    low = steps.floor()
    up = steps - low  # above a half, or at a half beside an odd integer: the integer above
    q = low + ((up > 0.5) | ((up == 0.5) & (low % 2 != 0)))
    return q * scale[:, None], scale


def exact(case, seed):
    st = prepare(case, seed)
    op, n, d, V, S, K, T = (case[k] for k in ("op", "n", "d", "V", "S", "K", "T"))
    with torch.no_grad():
        if op in ("logits", "train"):
            w = st["wq"].double() * st["w_scale"].double()[:, None]
            x = _exact_rows(st["rows"])[0]
            z = torch.cat([part @ w.T for part in x.split(1024)])
            if op == "logits":
                return z
            g = st["grad"].double()
            return {"logits": z, "grads": [g @ w, g.T.contiguous() @ x]}
        if op == "held":
            if not case["group"]:
                x, scale = _exact_rows(st["x"])
                return {"scale": scale, "x": x}
            xs, scales = zip(*(_exact_rows(part) for part in st["x"].split(case["group"], 1)))
            return {"scale": torch.stack(scales, 1), "x": torch.cat(xs, 1)}
        logp = torch.zeros(S, K + 1, dtype=torch.float64, device="cuda")
        tokens = torch.full((S, K + 1), -1, dtype=torch.int64, device="cuda")
        accepted = torch.zeros(S, dtype=torch.int64, device="cuda")
        drafts, lengths, u = st["drafts"].tolist(), st["lengths"].tolist(), st["uniform"].double().tolist()
        for s in range(S):
            target = torch.log_softmax(st["logits"][s].double() / T, 1)
            draft = None if st["draft_logits"] is None else torch.log_softmax(st["draft_logits"][s].double() / T, 1)
            best = st["logits"][s].double().cpu().numpy().argmax(1) if case["greedy"] else None
            i = 0
            while i < lengths[s]:
                v = drafts[s][i]
                if case["greedy"]:
                    ok = v == best[i]
                else:
                    ok = u[s][i] * (1.0 if draft is None else draft[i, v].exp().item()) < target[i, v].exp().item()
                if not ok:
                    break
                tokens[s, i], logp[s, i] = v, target[i, v]
                i += 1
            accepted[s] = i
            if case["greedy"]:
                v = int(best[i])
            else:
                mass = target[i].exp()
                if i < lengths[s]:
                    left = mass.clone()
                    if draft is None:
                        left[drafts[s][i]] = 0.0
                    else:
                        left = torch.relu(left - draft[i].exp())
                    mass = left if left.any() else mass
                steps = mass.cumsum(0)
                v = int(torch.searchsorted(steps, steps[-1:] * u[s][K], right=True)[0])
                v = min(v, int(mass.nonzero()[-1, 0]))
            tokens[s, i], logp[s, i] = v, target[i, v]
        return {"tokens": tokens, "accepted": accepted, "logp": logp}
