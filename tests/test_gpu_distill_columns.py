"""distill_columns and its gradient against the 64-bit oracle.

Tolerances. kl = sum q (log q - log p): log p as head_topk's (2e-5 at most), log q and q a softmax of K <= 256 values
(2^-22 relative each), so 4e-5 + 2^-21 sum q |log q - log p|. dz = g (Q p - w) / T: p is off by 2^-22 + 2^-24 |t| relative
(t = log2 p above -150: 2^-16), S's 1.2e-5 and Q and w by 2^-21, so 4e-5 of g (Q p + w) / T, and half a step of the
logits' type (f16 below its normal range: 2^-25)."""

import math

import pytest
import torch

from oracle import distill as odist

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _lists(n, V, K, seed, holes=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] if K <= V else torch.randint(0, V, (K,), generator=g)
                       for _ in range(n)])
    t = torch.randn(n, K, generator=g) * 2 - 4
    if holes:
        ids[torch.rand(n, K, generator=g) < 0.1] = -1
        ids[torch.rand(n, K, generator=g) < 0.05] = V  # past the vocabulary: empty as well
        t[torch.rand(n, K, generator=g) < 0.1] = -math.inf
        if n > 2:
            ids[1] = -1
            t[2] = -math.inf
    return ids, t


def _check(z, T, ids, t, g, normalise=True, view=None):
    from octopus_amd.distill_op import distill_columns

    dev = (z.cuda() if view is None else view(z)).detach().requires_grad_(True)
    kl = distill_columns(dev, T, ids.cuda(), t.cuda(), normalise=normalise)
    (grad,) = torch.autograd.grad(kl, dev, g.cuda())
    assert kl.dtype == torch.float32 and grad.dtype == z.dtype and grad.shape == z.shape
    s = z.double() / T
    want, dkl = odist.divergence(s, ids, t, normalise)
    q = odist.weights(ids, t, z.shape[1], normalise)
    lp = torch.log_softmax(s, 1).gather(1, ids.clamp(0, z.shape[1] - 1))
    scale = torch.where(q > 0, q * (torch.log(q).abs() + lp.abs()), torch.zeros_like(q)).sum(1)
    got = kl.detach().cpu().double()
    assert torch.equal(got.isfinite(), want.isfinite())
    ok = want.isfinite()
    Q = q.sum(1)
    assert ((got - want).abs()[ok] <= 4e-5 * Q[ok].clamp(min=1e-3) + 2 ** -21 * scale[ok]).all(), (got - want).abs().max()
    wg = dkl * g.double()[:, None] / T
    p = torch.softmax(s, 1)
    w = torch.zeros_like(p).scatter_add_(1, ids.clamp(0, z.shape[1] - 1), q)
    size = (g.double().abs() / T)[:, None] * (torch.where(Q[:, None] > 0, Q[:, None] * p, 0.0) + w)  # p may be NaN at Q 0
    tol = torch.finfo(z.dtype).eps / 2 * wg.abs() + 4e-5 * size + (2 ** -25 if z.dtype == torch.float16 else 1e-37)
    err = (grad.cpu().double() - wg).abs()
    assert (err <= tol).all(), ((err - tol).max(), err.max())
    return kl.detach(), grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (3, 5, 5), (4, 64, 3), (5, 1000, 64), (3, 4099, 256), (4, 32003, 20),
                                   (2, 151936, 64), (2, 128257, 100)])
@pytest.mark.parametrize("normalise", [True, False])
def test_sizes(dtype, n, V, K, normalise):
    g = torch.Generator().manual_seed(V + K)
    z = (torch.randn(n, V, generator=g) * 2.5).to(dtype)
    ids, t = _lists(n, V, K, V, holes=V > 8)
    _check(z, 1.0 if V % 2 else 0.7, ids, t, torch.rand(n, generator=g) + 0.1, normalise)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_in_several_slots(dtype):
    """Equal tokens in a list add their weights, in the divergence and in the gradient."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(4, 3000, generator=g).to(dtype)
    ids, t = _lists(4, 3000, 12, 2, holes=False)
    ids[0] = 77
    ids[1, [0, 5, 7]] = 2999
    ids[2, 3:] = ids[2, 0]
    ids[3, [0, 11]] = 0
    _check(z, 1.3, ids, t, torch.ones(4))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(dtype):
    """Student logits of -inf and of the type's lowest value, on and off the list; a listed token of probability 0 makes
    its row's divergence infinite and leaves its gradient -q."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(6)
    z = torch.randn(6, 2001, generator=g).to(dtype)
    ids, t = _lists(6, 2001, 9, 7, holes=False)
    z[0, 1000:] = -math.inf
    ids[0] = torch.arange(9)
    z[1, 1000:] = low
    ids[1] = torch.arange(9)
    z[2] = low
    z[3, ids[3, 0]] = -math.inf
    z[4] = -math.inf
    ids[4] = -1
    z[5] = math.nan
    t[5] = -math.inf
    _, grad = _check(z, 1.0, ids, t, torch.ones(6))
    assert (grad[4:] == 0).all()


def test_teacher_extremes():
    """Teacher values far apart and large; NaN stays NaN and in its row."""
    from octopus_amd.distill_op import distill_columns

    z = torch.randn(4, 500, generator=torch.Generator().manual_seed(8))
    ids = torch.arange(8).repeat(4, 1)
    t = torch.zeros(4, 8)
    t[0] = torch.tensor([0.0, -200.0, -1e30, 3e38 * 0, -50.0, -90.0, -104.0, -150.0])
    t[1] = 1e30
    t[2, 1:] = torch.finfo(torch.float32).min
    _check(z, 1.0, ids, t, torch.ones(4))
    t[3, 2] = math.nan
    kl = distill_columns(z.cuda(), 1.0, ids.cuda(), t.cuda())
    assert kl[3].isnan() and kl[:3].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Logits off a 16-byte boundary (their gradient is not: value by value) and with columns apart; strided lists."""
    g = torch.Generator().manual_seed(9)
    z = torch.randn(3, 1501, generator=g).to(dtype)
    ids, t = _lists(3, 1501, 10, 10)

    def odd(x):
        base = torch.zeros(3, 1600, dtype=dtype, device="cuda")
        base[:, 3:1504] = x.cuda()
        return base[:, 3:1504]

    a = _check(z, 1.0, ids, t, torch.ones(3), view=odd)
    b = _check(z, 1.0, ids, t, torch.ones(3), view=lambda x: x.T.contiguous().cuda().T)
    assert (a[0] - b[0]).abs().max() <= 4e-5  # the sums start at another boundary
    wide = torch.full((3, 20), -1)
    wide[:, ::2] = ids
    wt = torch.zeros(3, 20)
    wt[:, ::2] = t
    from octopus_amd.distill_op import distill_columns
    kl = distill_columns(z.cuda(), 1.0, wide.cuda()[:, ::2], wt.cuda()[:, ::2])
    assert torch.equal(kl, distill_columns(z.cuda(), 1.0, ids.cuda(), t.cuda()))
    assert torch.equal(kl, distill_columns(z.cuda(), 1.0, ids.int().cuda(), t.double().cuda()))


def test_gradient_against_differences():
    """fp32: the gradient against central differences of the 64-bit divergence."""
    from octopus_amd.distill_op import distill_columns

    z = torch.randn(2, 40, generator=torch.Generator().manual_seed(11))
    ids, t = _lists(2, 40, 6, 12)
    dev = z.cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(distill_columns(dev, 0.8, ids.cuda(), t.cuda()).sum(), dev)
    h = 1e-5
    for r in range(2):
        for v in range(40):
            up, dn = z.double().clone(), z.double().clone()
            up[r, v] += h
            dn[r, v] -= h
            d = (odist.divergence(up / 0.8, ids, t)[0][r] - odist.divergence(dn / 0.8, ids, t)[0][r]) / (2 * h)
            assert abs(grad[r, v].item() - d.item()) <= 1e-6  # fp32 2^-22, differences h^2 and 1e-16 / h


def test_many_rows():
    """More rows than a launch's grid takes in y: the last rows' gradients."""
    from octopus_amd.distill_op import distill_columns

    n, V = 65535 + 9, 16
    z = torch.randn(n, V, generator=torch.Generator().manual_seed(13)).cuda().requires_grad_(True)
    ids = torch.randint(0, V, (n, 2), device="cuda")
    t = torch.randn(n, 2, device="cuda")
    kl = distill_columns(z, 1.0, ids, t)
    (grad,) = torch.autograd.grad(kl.sum(), z)
    want, dkl = odist.divergence(z.detach()[-20:].cpu().double(), ids[-20:].cpu(), t[-20:].cpu())
    assert (kl[-20:].detach().cpu() - want).abs().max() <= 4e-5
    assert (grad[-20:].cpu() - dkl).abs().max() <= 4e-5


def test_graph_replays():
    from octopus_amd.distill_op import distill_columns_bwd, distill_columns_fwd

    z = torch.randn(5, 9000, device="cuda").to(torch.bfloat16)
    ids, t = (x.cuda() for x in _lists(5, 9000, 33, 14))
    g = torch.ones(5, device="cuda")

    def step():
        kl, state, q = distill_columns_fwd(z, ids, t, 1.0, False)
        return kl, distill_columns_bwd(z, ids, q, 1.0, state, g)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for s in range(3):
        z.copy_(torch.randn(5, 9000, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_refusals():
    from octopus_amd.distill_op import distill_columns

    z = torch.randn(3, 50, device="cuda")
    ids = torch.zeros(3, 4, dtype=torch.int64, device="cuda")
    t = torch.zeros(3, 4, device="cuda")
    wide = torch.zeros(3, 257, device="cuda")
    for bad in [(z, 0.0, ids, t), (z, 1.0, ids[:2], t[:2]), (z, 1.0, ids, t[:, :3]), (z, 1.0, ids[:, :0], t[:, :0]),
                (z, 1.0, wide.long(), wide), (z[0], 1.0, ids, t), (z, 1.0, ids.float(), t), (z, 1.0, ids.cpu(), t)]:
        with pytest.raises(ValueError):
            distill_columns(*bad)
    with pytest.raises(NotImplementedError):
        distill_columns(z.double(), 1.0, ids, t)
    assert distill_columns(z[:0], 1.0, ids[:0], t[:0]).shape == (0,)
