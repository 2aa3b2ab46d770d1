"""The oracles of the lists, the divergence and the embedding against something other than their own formulas: torch's
top-k, softmax, KL divergence, embedding and autograd, in 64 bits, and closed forms."""

import math

import pytest
import torch

from oracle import distill, embed


def _lists(n, V, K, seed, empty=0.3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(-2, V + 2, (n, K), generator=g)
    t = torch.randn(n, K, generator=g, dtype=torch.float64)
    t[torch.rand(n, K, generator=g) < empty] = -math.inf
    ids[0] = -1  # a row without a slot
    ids[1] = ids[1, 0].clamp(0, V - 1)  # one token in every slot
    return ids, t


def test_topk_against_torch():
    z = torch.randn(9, 77, generator=torch.Generator().manual_seed(0), dtype=torch.float64)  # no two equal
    ids, logp = distill.topk(z, 0.7, 12)
    want = torch.topk(z, 12, dim=1)
    assert torch.equal(ids, want.indices)
    assert torch.allclose(logp, torch.log_softmax(z / 0.7, 1).gather(1, want.indices), rtol=0, atol=1e-14)


def test_topk_of_equal_values():
    z = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 3.0, 0.0, -0.0]])
    assert distill.topk(z, 1.0, 7)[0].tolist() == [[1, 2, 4, 0, 5, 6, 3]]
    z[0, 5] = math.nan
    assert distill.topk(z, 1.0, 3)[0].tolist() == [[5, 1, 2]]


@pytest.mark.parametrize("normalise", [True, False])
def test_divergence_against_dense_distributions(normalise):
    """The lists as distributions over the whole vocabulary: torch.kl_div's sums and autograd's gradient."""
    n, V, K = 8, 23, 6
    ids, t = _lists(n, V, K, 1)
    s = torch.randn(n, V, generator=torch.Generator().manual_seed(2), dtype=torch.float64, requires_grad=True)
    kl, grad = distill.divergence(s.detach(), ids, t, normalise)
    used = (ids >= 0) & (ids < V) & (t > -math.inf)
    q = torch.where(used, t.masked_fill(~used, -math.inf).exp(), torch.zeros(()).double())
    if normalise:
        q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
    assert torch.allclose(distill.weights(ids, t, V, normalise), q, rtol=1e-13, atol=0)
    dense = torch.zeros(n, V, dtype=torch.float64).scatter_add_(1, ids.clamp(0, V - 1), q)
    # slot by slot sum q log q, where kl_div has the tokens' merged weights
    cross = torch.nn.functional.kl_div(torch.log_softmax(s, 1), dense, reduction="none").sum(1)
    want = cross - torch.special.xlogy(dense, dense).sum(1) + torch.special.xlogy(q, q).sum(1)
    assert torch.allclose(kl, want.detach(), rtol=0, atol=1e-13)
    got, = torch.autograd.grad(want.sum(), s)
    assert torch.allclose(grad, got, rtol=0, atol=1e-13)
    assert kl[0] == 0 and not grad[0].any()


def test_divergence_from_itself():
    """The whole vocabulary listed with the student's own log-probabilities: 0, and no gradient."""
    s = torch.randn(3, 11, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    kl, grad = distill.divergence(s, torch.arange(11).expand(3, 11), torch.log_softmax(s, 1))
    assert kl.abs().max() < 1e-14 and grad.abs().max() < 1e-15


@pytest.mark.parametrize("padding_idx", [None, 4])
def test_embedding_against_torch(padding_idx):
    g = torch.Generator().manual_seed(4)
    w = torch.randn(9, 5, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, 9, (3, 7), generator=g)
    up = torch.randn(3, 7, 5, generator=g, dtype=torch.float64)
    out = torch.nn.functional.embedding(ids, w, padding_idx=padding_idx) * 1.5
    assert torch.equal(embed.lookup(w.detach(), ids, 1.5), out.detach())
    want, = torch.autograd.grad(out, w, up)
    got, mag, cnt = embed.gradient(up, ids, 9, 1.5, padding_idx)
    assert torch.allclose(got, want, rtol=0, atol=1e-14)
    keep = torch.ones(9, dtype=torch.bool)
    if padding_idx is not None:
        keep[padding_idx] = False
    assert torch.equal(cnt, torch.bincount(ids.flatten(), minlength=9) * keep) and (mag >= got.abs() - 1e-14).all()


def test_embedding_outside_the_vocabulary():
    ids = torch.tensor([-1, 3, 2])
    w = torch.ones(3, 2, dtype=torch.float64)
    assert embed.lookup(w, ids, 2.0).tolist() == [[0, 0], [0, 0], [2, 2]]
    assert embed.gradient(torch.ones(3, 2), ids, 3, 2.0)[0].tolist() == [[0, 0], [0, 0], [2, 2]]
