"""The operators together, as a distillation step uses them: the teacher's logits become lists, the student looks its tokens
up in W, a small mixing layer makes hidden rows, the head multiplies with the same W, and both ends' gradients meet in it."""

import pytest
import torch

from oracle import distill as odist
from oracle import embed as oemb

pytestmark = pytest.mark.gpu


def _batch(n, d, V, seed):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, d, generator=g) * 0.25).to(torch.bfloat16)
    mix = (torch.randn(d, d, generator=g) / d ** 0.5).to(torch.bfloat16)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[::17] = -1  # the packing between sequences
    teacher = (torch.randn(n, V, generator=g) * 2).to(torch.bfloat16)
    return w, mix, ids, teacher


def _student(w, mix, ids, teacher, K, scale, T, later=None):
    """(loss, the gradient of W, tokens and values of the lists); later: both ends' gradients added by hand."""
    from octopus_amd.distill_op import fused_distill_head, head_topk
    from octopus_amd.embed_op import embed_grad_add_, embed_rows
    from octopus_amd.head_op import compact_rows

    idx, count = compact_rows(ids >= 0)
    top, logp = head_topk(teacher, T, K)
    share = torch.full(ids.shape, 1.0 / ids.numel(), device=ids.device)
    if later is None:
        leaf = w.detach().clone().requires_grad_(True)
        x = embed_rows(leaf, ids, scale)
        h = torch.matmul(x, mix)
        loss, _ = fused_distill_head(h, leaf, top, logp, T, share, idx=idx, count=count)
        loss.backward()
        return loss.detach(), leaf.grad, top, logp
    head = w.detach().clone().requires_grad_(True)
    x = embed_rows(w, ids, scale).requires_grad_(True)
    h = torch.matmul(x, mix)
    loss, _ = fused_distill_head(h, head, top, logp, T, share, idx=idx, count=count)
    loss.backward()
    return loss.detach(), embed_grad_add_(head.grad, x.grad, ids, scale), top, logp


@pytest.mark.parametrize("n,d,V,K", [(40, 64, 700, 8), (300, 128, 3001, 40)])
def test_a_step_of_a_tied_student(n, d, V, K):
    """Against the step in 64 bits from the same 16-bit roundings of x, h and their gradients; the gradient of W by autograd
    (two dense gradients added) and with the lookup's added in place to the head's."""
    w, mix, ids, teacher = _batch(n, d, V, n)
    scale, T = 1.5, 0.8
    dev = [t.cuda() for t in (w, mix, ids, teacher)]
    loss, gw, top, logp = _student(*dev, K, scale, T)
    loss2, gw2, _, _ = _student(*dev, K, scale, T, later=True)
    want_ids, want_logp = odist.topk(teacher, T, K)
    assert torch.equal(top.cpu(), want_ids) and (logp.cpu() - want_logp).abs().max() <= 4e-5

    x = oemb.lookup(w, ids, scale).to(torch.bfloat16).double()
    h = (x @ mix.double()).to(torch.bfloat16).double()
    on = ids >= 0
    s = h @ w.double().T / T
    kl, dkl = odist.divergence(s, torch.where(on[:, None], want_ids, -1), want_logp)
    dz = dkl / n / T
    want = (kl / n)[on].sum()
    # h's rounding may fall the other way where the product's own sum differs: 2^-8 of a logit's terms, at random signs
    assert abs(loss.item() - want.item()) <= 2e-2 * want.item()
    head = dz.T @ h
    gx = (dz @ w.double()) @ mix.double().T
    emb, _, _ = oemb.gradient(gx, ids, V, scale)
    total = head + emb
    # each end's gradient lies within the 1e-2 (relative norm) of 16-bit gradients; x's passes one more 16-bit product
    for got in (gw, gw2):
        assert (got.cpu().double() - total).norm() <= 1e-2 * head.norm() + 2e-2 * emb.norm()
    assert loss == loss2
    # the same two gradients, added after one rounding each or after one
    assert (gw.float() - gw2.float()).norm() <= 2 ** -8 * (gw.float().norm() + head.norm() + emb.norm())


def test_the_step_replayed_from_a_graph():
    """Captured after a warm-up whose own graph of autograd is gone; other tokens and logits in place at each replay."""
    from octopus_amd.distill_op import head_step_distill, head_topk
    from octopus_amd.embed_op import embed_bwd, embed_rows

    w, mix, ids, teacher = (t.cuda() for t in _batch(60, 64, 900, 5))

    def step():
        top, logp = head_topk(teacher, 1.0, 16)
        x = embed_rows(w, ids, 2.0)
        h = torch.matmul(x, mix)
        loss, kl, gh, gw = head_step_distill(h, w, None, top, logp, None, None, None, 1.0, 1.0, 1.0, False, False, True,
                                             True)
        return loss, kl, gw, embed_bwd(torch.matmul(gh, mix.T.contiguous()), ids, 900, 2.0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for s in range(3):
        g = torch.Generator().manual_seed(s)
        ids.copy_(torch.randint(0, 900, (60,), generator=g))
        teacher.copy_((torch.randn(60, 900, generator=g) * 2).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_two_streams_at_once():
    """Two steps of other inputs queued on two streams before either is waited for: each as alone."""
    one, two = ([t.cuda() for t in _batch(200, 128, 2000, s)] for s in (6, 7))
    want = [_student(*x, 20, 1.0, 1.0)[:2] for x in (one, two)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for x, st in zip((one, two), streams):
        with torch.cuda.stream(st):
            got.append(_student(*x, 20, 1.0, 1.0)[:2])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
