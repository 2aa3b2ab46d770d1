"""The embedding lookup and its gradient by sorted tokens against the 64-bit oracle.

Tolerances: the lookup rounds one fp32 product (2^-24) to the type (eps / 2). The gradient sums up to c tokens of an entry
in fp32 (c + 2 roundings of 2^-24 of the magnitudes' sum) and rounds once."""

import pytest
import torch

from oracle import embed as oemb

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return 2 ** -25 if dtype == torch.float16 else 1e-40


def _tokens(n, V, seed, hot=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[torch.rand(n, generator=g) < hot] = V // 2  # one entry takes this share
    return ids


def _check_gradient(grad, ids, V, scale, got, dtype, old=None, padding=None):
    want, mag, cnt = oemb.gradient(grad, ids, V, scale, padding)
    if old is not None:
        want, mag = want + old.double(), mag + old.double().abs()
    tol = (_half(dtype) * want.abs() + (cnt[:, None] + 4) * 2 ** -24 * mag) * (1 + 2 ** -8) + _tiny(dtype)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), (err - tol).max()
    none = cnt == 0
    assert torch.equal(got.cpu()[none], torch.zeros_like(got.cpu()[none]) if old is None else old[none])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 50, 8), (5, 7, 24), (16, 1000, 4096), (33, 300, 1023), (300, 5000, 1024),
                                   (65, 40, 2305)])
def test_lookup(dtype, n, V, d):
    from octopus_amd.embed_op import embed_rows

    g = torch.Generator().manual_seed(n + V)
    w = torch.randn(V, d, generator=g).to(dtype)
    ids = _tokens(n, V, n)
    if n > 4:
        ids[[0, n - 1]] = torch.tensor([-1, V])
        ids[2] = -2 ** 40
    scale = d ** 0.5
    got = embed_rows(w.cuda(), ids.cuda(), scale)
    want = oemb.lookup(w, ids, scale)
    assert got.dtype == dtype and got.shape == (n, d)
    tol = (_half(dtype) + 2 ** -23) * want.abs() + _tiny(dtype)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(embed_rows(w.cuda(), ids.cuda()).cpu().double(), oemb.lookup(w, ids, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,d,hot", [(1, 1, 1, 0), (1, 600, 8, 0), (31, 50, 24, 0), (32, 3, 8, 0), (33, 1, 520, 0),
                                       (200, 2000, 1031, 0.3), (700, 513, 64, 0.9), (1000, 512, 16, 0.0),
                                       (1500, 1025, 512, 0.5), (4096, 300, 40, 1.0), (5000, 70000, 8, 0.02)])
def test_gradient(dtype, n, V, d, hot):
    """Entries of one token and of thousands, that end at, before and behind a piece's border; one entry alone."""
    from octopus_amd.embed_op import embed_rows

    g = torch.Generator().manual_seed(n * d)
    w = torch.zeros(V, d, dtype=dtype, device="cuda", requires_grad=True)
    ids = _tokens(n, V, n + 1, hot)
    if n > 40:
        ids[3], ids[17], ids[n - 1] = -1, V, 2 ** 33  # no entry's
    grad = torch.randn(n, d, generator=g).to(dtype)
    (got,) = torch.autograd.grad(embed_rows(w, ids.cuda(), 1.7), w, grad.cuda())
    assert got.dtype == dtype and got.shape == (V, d)
    scale = torch.tensor(1.7, dtype=torch.float32).item()
    _check_gradient(grad, ids, V, scale, got, dtype)
    (again,) = torch.autograd.grad(embed_rows(w, ids.cuda(), 1.7), w, grad.cuda())
    assert torch.equal(got, again)


@pytest.mark.parametrize("gdt,wdt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                     (torch.float16, torch.float32), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("d", [128, 131])
def test_gradient_of_other_types_and_padding(gdt, wdt, d):
    from octopus_amd.embed_op import embed_bwd

    n, V = 300, 90
    grad = torch.randn(n, d, generator=torch.Generator().manual_seed(d)).to(gdt)
    ids = _tokens(n, V, 5, 0.4)
    got = embed_bwd(grad.cuda(), ids.cuda(), V, -0.5, padding_idx=45, dtype=wdt)
    _check_gradient(grad, ids, V, -0.5, got, wdt, padding=45)
    assert torch.equal(got, embed_bwd(grad.cuda(), ids.int().cuda(), V, -0.5, padding_idx=45 - V, dtype=wdt))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,d,hot", [(1, 9, 8, 0), (300, 2000, 96, 0.4), (257, 40, 77, 0.1)])
def test_add_in_place(dtype, n, V, d, hot):
    """The rows of the tokens get their sums on top; the others stay as they are, bit for bit (a NaN among them)."""
    from octopus_amd.embed_op import embed_grad_add_

    g = torch.Generator().manual_seed(n)
    ids = _tokens(n, V - 1, n, hot)  # the last entry never occurs
    grad = torch.randn(n, d, generator=g).to(dtype)
    old = torch.randn(V, d, generator=g).to(dtype)
    into = torch.zeros(V, d + 24, dtype=dtype, device="cuda")
    into[:, :d] = old.cuda()
    got = embed_grad_add_(into[:, :d], grad.cuda(), ids.cuda(), 0.25)
    _check_gradient(grad, ids, V, 0.25, got, dtype, old=old)
    assert (into[:, d:] == 0).all()
    into[V - 1, 0] = float("nan")
    embed_grad_add_(into[:, :d], grad.cuda(), ids.cuda(), 0.25)
    assert into[V - 1, 0].isnan() and into[:V - 1].isfinite().all()


def test_views():
    """Strided weights, strided and expanded gradients, ids of two dimensions, no tokens at all."""
    from octopus_amd.embed_op import embed_bwd, embed_grad_add_, embed_rows

    w = torch.randn(50, 100, device="cuda")
    ids = torch.randint(0, 50, (4, 6), device="cuda")
    sub = w[:, 3:67]
    assert torch.equal(embed_rows(sub, ids), sub[ids]) and embed_rows(w.T, ids).shape == (4, 6, 50)
    assert torch.equal(embed_rows(w.T, ids), w.T[ids])
    leaf = w.clone().requires_grad_(True)
    embed_rows(leaf, ids, 2.0).sum().backward()  # an expanded gradient
    assert torch.equal(leaf.grad, 2.0 * torch.bincount(ids.reshape(-1), minlength=50)[:, None].expand(50, 100).float())
    grad = torch.randn(4, 6, 140, device="cuda")[:, :, 20:84]
    a, b = embed_bwd(grad, ids, 50), embed_bwd(grad.contiguous(), ids, 50)
    assert torch.equal(a, b)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert embed_rows(w, none).shape == (0, 100)
    assert (embed_bwd(torch.empty(0, 100, device="cuda"), none, 50) == 0).all()
    assert torch.equal(embed_grad_add_(w.clone(), torch.empty(0, 100, device="cuda"), none), w)
    out = torch.full((6,), -1, device="cuda")
    assert (embed_rows(w, out) == 0).all() and (embed_bwd(torch.ones(6, 8, device="cuda"), out, 9) == 0).all()


def test_graph_replays():
    """Other tokens in place between replays of a captured gradient, and an addition into a kept one."""
    from octopus_amd.embed_op import embed_bwd, embed_grad_add_, embed_rows

    V, n, d = 700, 400, 264
    ids = torch.randint(0, V, (n,), device="cuda")
    grad = torch.randn(n, d, device="cuda").to(torch.bfloat16)
    w = torch.randn(V, d, device="cuda").to(torch.bfloat16)
    into = torch.zeros(V, d, device="cuda")

    def step():
        return embed_rows(w, ids, 3.0), embed_bwd(grad, ids, V, 3.0)

    step()
    embed_grad_add_(into, grad, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
        embed_grad_add_(into, grad, ids)
    for s in range(3):
        ids.copy_(torch.randint(0, V // (s + 1), (n,), generator=torch.Generator().manual_seed(s)))
        into.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
        assert torch.equal(into, embed_grad_add_(torch.zeros_like(into), grad, ids))


def test_refusals():
    from octopus_amd.embed_op import embed_bwd, embed_grad_add_, embed_rows

    w = torch.randn(20, 16, device="cuda")
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    g = torch.randn(5, 16, device="cuda")
    for call in [lambda: embed_rows(w[0], ids), lambda: embed_rows(w, ids.float()), lambda: embed_rows(w, ids.cpu()),
                 lambda: embed_rows(w[:0], ids), lambda: embed_rows(w, ids, padding_idx=20),
                 lambda: embed_bwd(g, ids[:4], 20), lambda: embed_bwd(g, ids, 0), lambda: embed_bwd(g[:, :0], ids, 20),
                 lambda: embed_grad_add_(w.T, torch.randn(5, 20, device="cuda"), ids),
                 lambda: embed_grad_add_(w, g[:, :8], ids)]:
        with pytest.raises((ValueError, RuntimeError)):
            call()
    for call in [lambda: embed_rows(w.double(), ids), lambda: embed_bwd(g.double(), ids, 20),
                 lambda: embed_grad_add_(w.double(), g, ids)]:
        with pytest.raises(NotImplementedError):
            call()
