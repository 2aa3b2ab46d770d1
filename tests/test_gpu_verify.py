"""Verification of drafted tokens (octopus_amd.verify_op) on the GPU against the definition in 64 bits."""

import math

import pytest
import torch

from octopus_amd import verify_op
from oracle import verify as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
NINF = -math.inf


def _inputs(S, K, V, dtype, seed=0, apart=0.7):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(S, K + 1, V, generator=g) * 2.5
    zd = z[:, :K] + apart * torch.randn(S, K, V, generator=g)
    z, zd = z.to(dtype), zd.to(dtype)
    x = torch.multinomial(torch.softmax(zd.float(), 2).reshape(S * K, V), 1, generator=g).view(S, K) if K else \
        torch.empty(S, 0, dtype=torch.int64)
    return z, zd, x, torch.rand(S, K + 1, generator=g)


def _check(z, x, u, T=1.0, zd=None, lengths=None, greedy=False):
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    tokens, accepted, logp = verify_op.verify_drafts(d(z), d(x), d(u), T, draft_logits=d(zd), lengths=d(lengths),
                                                     greedy=greedy)
    want, count, lp = oracle.verify(z, x, u, T, zd, lengths, greedy)
    assert tokens.dtype == accepted.dtype == torch.int64 and logp.dtype == torch.float32
    assert accepted.tolist() == count
    assert tokens.tolist() == want
    lp = torch.tensor(lp, dtype=torch.float64).view(logp.shape)
    # 64-bit arithmetic, rounded to fp32 once: 2^-24, and 1e-12 for what 64 bits lose
    torch.testing.assert_close(logp.cpu().double(), lp, rtol=2.0 ** -24 + 1e-12, atol=1e-12, equal_nan=True)
    return tokens.cpu(), accepted.cpu()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,K,V", [(1, 4, 1000), (3, 1, 1), (5, 2, 7), (4, 3, 4096), (3, 5, 4097), (2, 2, 9001), (9, 0, 513),
                                   (2, 63, 130), (1, 4, 20001)])
def test_drafts(S, K, V, dtype):
    z, zd, x, u = _inputs(S, K, V, dtype, S + V)
    for T in (1.0, 0.7):
        _check(z, x, u, T, zd)
    _check(z, x, u, 1.3)
    _check(z, x, u, greedy=True)


def test_lengths():
    z, zd, x, u = _inputs(8, 3, 300, torch.bfloat16, apart=0.05)
    n = torch.tensor([0, 1, 2, 3, 4, 100, -1, 2])
    for dtype in (torch.int64, torch.int32):
        _, acc = _check(z, x, u, 1.0, zd, n.to(dtype))
        assert (acc <= n.clamp(0, 3)).all()
    # what lies behind a sequence's length is not looked at
    z2, zd2, x2 = z.clone(), zd.clone(), x.clone()
    for s, k in enumerate(n.clamp(0, 3).tolist()):
        z2[s, k + 1:] = math.nan
        zd2[s, k:] = math.nan
        x2[s, k:] = 10 ** 9
    a = verify_op.verify_drafts(z.to(DEV), x.to(DEV), u.to(DEV), 1.0, draft_logits=zd.to(DEV), lengths=n.to(DEV))
    b = verify_op.verify_drafts(z2.to(DEV), x2.to(DEV), u.to(DEV), 1.0, draft_logits=zd2.to(DEV), lengths=n.to(DEV))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_masks(dtype):
    z, zd, x, u = _inputs(8, 2, 5000, dtype, 3)
    low = torch.finfo(dtype).min
    z[0, :, 10:] = NINF
    zd[0, :, 10:] = NINF
    x[0] = 3
    z[1, :, :4990] = low                      # the type's lowest value
    z[2] = low                                # nothing else: every token alike
    z[3, 0] = NINF                            # no distribution
    z[4, 1, 77] = math.nan
    z[5, 0, 4999] = math.inf
    zd[6, 0] = NINF                           # a draft that came from nowhere
    zd[7, 0, 5] = math.nan
    tokens, acc = _check(z, x, u, 0.5, zd)
    assert tokens[3, 0] == -1 and tokens[5, 0] == -1 and acc[3] == acc[5] == acc[6] == acc[7] == 0
    assert tokens[6, 0] >= 0 and tokens[7, 0] >= 0
    _check(z, x, u, 0.5)
    _check(z, x, u, 0.5, greedy=True)


def test_drafts_outside_the_vocabulary():
    z, zd, x, u = _inputs(6, 2, 100, torch.float32)
    x[0, 0], x[1, 0], x[2, 1], x[3, 0] = -1, 100, 2 ** 40, -2 ** 62
    tokens, acc = _check(z, x, u, 1.0, zd)
    assert acc[0] == acc[1] == acc[3] == 0 and acc[2] <= 1
    _check(z, x, u)
    _check(z, x, u, greedy=True)


def test_numbers_at_the_borders():
    """Even distributions have running sums that 64 bits hold exactly: a number at one of them takes the token behind."""
    S, V = 64, 64
    z = torch.zeros(S, 1, V)
    u = (torch.arange(S).float() / V)[:, None]
    tokens, _ = _check(z, torch.empty(S, 0, dtype=torch.int64), u)
    assert tokens[:, 0].tolist() == list(range(V))
    below = (u.view(torch.int32) - 1).clamp_min(0).view(torch.float32)
    tokens, _ = _check(z, torch.empty(S, 0, dtype=torch.int64), below)
    assert tokens[:, 0].tolist() == [0] + list(range(V - 1))
    # u q = p is not accepted
    zd = torch.zeros(2, 1, V)
    z = torch.zeros(2, 2, V)
    z[:, 0, 0] = math.log(2.0)
    tokens, acc = verify_op.verify_drafts(zd.expand(2, 2, V).contiguous().to(DEV), torch.zeros(2, 1, dtype=torch.int64,
                                          device=DEV), torch.tensor([[1.0, 0.5], [0.99999994, 0.5]], device=DEV), 1.0,
                                          draft_logits=zd.to(DEV))[:2]
    assert acc.tolist() == [0, 1] and tokens[0].tolist() == [V // 2, -1]
    # numbers that are none: a last token, or nothing
    z, zd, x, _ = _inputs(4, 1, 50, torch.float32)
    u = torch.tensor([[0.0, 0.0], [1.0, 1.0], [2.0, 0.3], [0.0, 1.0]])
    _check(z, x, u, 1.0, zd)
    u[0, 1] = math.nan
    got = verify_op.verify_drafts(z.to(DEV), x.to(DEV), u.to(DEV), 1.0)[0]
    assert got[0, 1 if got[0, 0] == x[0, 0] else 0].item() == oracle.verify(z, x, u, 1.0)[0][0][1]


def test_equal_models_accept_everything():
    z, _, x, u = _inputs(16, 4, 2000, torch.bfloat16)
    _, acc = _check(z, x, u, 0.9, z[:, :4].clone())
    assert (acc == 4).all()


def test_the_last_of_many_equal_maxima():
    z = torch.zeros(3, 2, 9000, dtype=torch.float16)
    z[0, 0, 8000] = 1
    z[1, :, 4095:4098] = 2
    x = torch.tensor([[8000], [4095], [1]])
    tokens, acc = _check(z, x, None, greedy=True)
    assert acc.tolist() == [1, 1, 0] and tokens[2, 0] == 0


def test_strides():
    z, zd, x, u = _inputs(5, 3, 203, torch.bfloat16)
    wide = torch.full((5, 4, 210), NINF, dtype=torch.bfloat16, device=DEV)
    wide[:, :, 3:206] = z.to(DEV)
    wd = torch.full((3, 5, 207), NINF, dtype=torch.bfloat16, device=DEV)
    wd[:, :, 1:204] = zd.transpose(0, 1).to(DEV)
    want = verify_op.verify_drafts(z.to(DEV), x.to(DEV), u.to(DEV), 1.0, draft_logits=zd.to(DEV))
    for target in (wide[:, :, 3:206], z.to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = verify_op.verify_drafts(target, x.to(DEV).t().contiguous().t(), u.to(DEV).t().contiguous().t(), 1.0,
                                      draft_logits=wd.transpose(0, 1)[:, :, 1:204])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = verify_op.verify_drafts(z[:1].to(DEV).expand(4, 4, 203), x[:1].to(DEV).expand(4, 3), u[:1].to(DEV).expand(4, 4),
                                  1.0)
    assert (one[0] == one[0][:1]).all()


# ---- many logits: the rows' sums with 32-bit exponentials first -------------------------------------------------------

def _check_many(z, x, u, T=1.0, zd=None, lengths=None):
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    assert z.numel() + (0 if zd is None else zd.numel()) >= 1 << 24
    tokens, accepted, logp = verify_op.verify_drafts(d(z), d(x), d(u), T, draft_logits=d(zd), lengths=d(lengths))
    want, count, lp = oracle.verify_dense(z, x, u, T, zd, lengths)
    assert torch.equal(accepted.cpu(), count) and torch.equal(tokens.cpu(), want)
    # the accepted drafts' by a row sum that 32-bit exponentials make, within 4e-6 of it
    torch.testing.assert_close(logp.cpu().double(), lp, rtol=2.0 ** -24, atol=4e-6)
    return tokens.cpu(), accepted.cpu()


@pytest.mark.parametrize("dtype,S,K,V,T", [(torch.bfloat16, 40, 3, 61003, 1.0), (torch.float16, 300, 0, 56000, 0.7),
                                           (torch.float32, 9, 7, 128257, 1.3), (torch.bfloat16, 1030, 1, 5500, 1.0),
                                           (torch.bfloat16, 3, 1, 3000001, 0.9)])
def test_many_logits(dtype, S, K, V, T):
    z, zd, x, u = _inputs(S, K, V, dtype, S)
    n = torch.randint(0, K + 1, (S,), generator=torch.Generator().manual_seed(1))
    _check_many(z, x, u, T, zd if K else None)
    z[S // 2, :, 60:], zd[S // 2, :, 60:], x[S // 2] = NINF, NINF, 7
    _check_many(z, x, u, T, zd if K else None, n)
    if K and z.numel() >= 1 << 24:
        _check_many(z, x, u, T)


@pytest.mark.parametrize("sampled", [True, False])
def test_many_drafts_on_the_border(sampled):
    """u the number of 32 bits next to p / q: below, accepted, above, rejected, 2^-25 of it or less to decide by."""
    S, K, V = 150, 2, 40000
    z, zd, x, u = _inputs(S, K, V, torch.bfloat16, 5)
    zd = zd if sampled else None
    p = torch.log_softmax(z[:, :K].double(), 2).gather(2, x[:, :, None])[:, :, 0]
    q = torch.log_softmax(zd.double(), 2).gather(2, x[:, :, None])[:, :, 0] if sampled else torch.zeros_like(p)
    ratio = (p - q).exp()
    near = ratio.float()
    step = torch.where(near.double() < ratio, near, torch.nextafter(near, torch.zeros_like(near)))  # the largest below
    above = torch.nextafter(step, torch.full_like(step, 9.0))
    up = torch.rand(S, K, generator=torch.Generator().manual_seed(2)) < 0.4
    apart = (above.double() - ratio).abs() > 1e-12 * ratio
    u[:, :K] = torch.where(up & apart, above, step)
    _, acc = _check_many(z, x, u, 1.0, zd)
    assert torch.equal(acc, (~(up & apart)).long().cumprod(1).sum(1))


@pytest.mark.parametrize("noise", [3e-2, 1e-3, 1e-5])
def test_many_with_models_alike(noise):
    """Draft and target all but equal, rejected by numbers near 1: what is left of p - q is little, and in much of the
    vocabulary the two lie within 2^-15 of each other."""
    S, K, V = 90, 2, 40000
    z, _, x, u = _inputs(S, K, V, torch.float32, 6)
    g = torch.Generator().manual_seed(7)
    zd = z[:, :K] + noise * torch.randn(S, K, V, generator=g)
    zd[:, :, V // 2:] = z[:, :K, V // 2:]     # and exactly equal in half of it
    u[:, :K] = 1.0 - 2.0 ** -24
    _, acc = _check_many(z, x, u, 1.0, zd)
    assert (acc < K).any()


def test_many_without_a_distribution():
    z, zd, x, u = _inputs(700, 1, 13000, torch.bfloat16, 8)
    z[0, 0], z[1, 0, 12999], z[2, 0, 0] = NINF, math.nan, math.inf
    zd[3, 0], zd[4, 0, 1], x[5, 0] = NINF, math.inf, -1
    z[6] = torch.finfo(torch.bfloat16).min
    tokens, acc, logp = verify_op.verify_drafts(z.to(DEV), x.to(DEV), u.to(DEV), 1.0, draft_logits=zd.to(DEV))
    assert acc[:6].tolist() == [0] * 6 and tokens[:3].tolist() == [[-1, -1]] * 3 and torch.isnan(logp[:3, 0]).all()
    assert (logp[:6, 1] == 0).all() and (tokens[:6, 1] == -1).all()
    want, count, lp = oracle.verify_dense(z[3:6, 0:1], x[3:6, :0], u[3:6, 1:], 1.0)  # drawn from the target alone
    assert tokens[3:6, 0].tolist() == want[:, 0].tolist()
    want, count, _ = oracle.verify_dense(z[6:], x[6:], u[6:], 1.0, zd[6:])
    assert torch.equal(tokens[6:].cpu(), want) and torch.equal(acc[6:].cpu(), count)
    got = verify_op.verify_drafts(z.to(DEV), x.to(DEV), None, 1.0, greedy=True)
    assert got[0][:3].tolist() == [[-1, -1]] * 3
    best = z[7:].float().argmax(2)
    assert torch.equal(got[1][7:].cpu(), (x[7:, 0] == best[:, 0]).long())


def test_extreme_temperatures():
    z, zd, x, u = _inputs(3, 2, 200, torch.float32)
    for T in (1e-13, 1e-3, 1e4, 1e13):
        _check(z, x, u, T)
    z, zd, x, u = _inputs(700, 1, 13000, torch.float32)
    z[::3, :, ::2] = NINF
    x.clamp_(1, 12999).bitwise_or_(1)
    for T in (1e-13, 1e-5, 1e13):
        _check_many(z, x, u, T)


def test_refusals():
    z, zd, x, u = (t.to(DEV) for t in _inputs(3, 2, 50, torch.bfloat16))
    ok = dict(draft_logits=zd)
    for args, kw in [((z[0], x, u, 1.0), ok), ((z, x[:, :1], u, 1.0), ok), ((z, x, u[:, :2], 1.0), ok),
                     ((z, x, u.double(), 1.0), ok), ((z, x, None, 1.0), ok), ((z, x, u, 0.0), ok),
                     ((z, x, u, float("nan")), ok), ((z, x, u, 1e-39), ok), ((z, x.float(), u, 1.0), ok),
                     ((z, x, u, 1.0), dict(draft_logits=zd[:, :1])), ((z, x, u, 1.0), dict(draft_logits=zd.float())),
                     ((z, x, u, 1.0), dict(lengths=torch.ones(2, dtype=torch.int64, device=DEV))),
                     ((z, x.cpu(), u, 1.0), ok), ((z.cpu(), x, u, 1.0), {}), ((z[:, :, :0], x, u, 1.0), {})]:
        with pytest.raises(ValueError):
            verify_op.verify_drafts(*args, **kw)
    with pytest.raises(NotImplementedError):
        verify_op.verify_drafts(z.double(), x, u, 1.0)
    big = torch.zeros(1, 65, 10, device=DEV)
    with pytest.raises(ValueError):
        verify_op.verify_drafts(big, torch.zeros(1, 64, dtype=torch.int64, device=DEV), torch.zeros(1, 65, device=DEV), 1.0)
    empty = verify_op.verify_drafts(z[:0], x[:0], u[:0], 1.0, draft_logits=zd[:0])
    assert empty[0].shape == (0, 3) and empty[1].shape == (0,)
