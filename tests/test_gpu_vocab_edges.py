"""Calls of the lists, the distillation and the embedding at the edges of what their documentation allows."""

import pytest
import torch

from oracle import distill as odist

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("later", [False, True])
def test_a_soft_cap_of_negative_slope_keeps_the_roundings(later, monkeypatch):
    """z = 30 tanh(-x / 30): the weight gradient of bf16 operands takes two roundings of half a step each, the listed
    values' and the result's, as with a positive slope. Roundings of one size add in squares, so its error lies below
    sqrt(2.5) times the one that the exact gradient's own rounding costs; a third (h^T times a scale that is not a power of
    two) would bring it to sqrt(3)."""
    from octopus_amd import distill_op, head_op
    from octopus_amd.head_op import Post

    n, d, V, K, cap = 300, 256, 8192, 64, 30.0
    g = torch.Generator().manual_seed(21)
    h, w = torch.randn(n, d, generator=g).to(torch.bfloat16), (torch.randn(V, d, generator=g) * 0.02).to(torch.bfloat16)
    ids, t = torch.randint(0, V, (n, K), generator=g), torch.randn(n, K, generator=g)
    rw = torch.rand(n, generator=g) + 0.5
    monkeypatch.setattr(head_op, "_LATER_SHARE", 1 << 20)
    monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 0 if later else 1 << 62)
    monkeypatch.setattr(head_op, "_LATER_WORK", 1 << 62)
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    assert (distill_op._later_bytes(hd, wd, None, True, True) > 0) == later
    loss, kl = distill_op.fused_distill_head(hd, wd, ids.cuda(), t.cuda(), 1.0, rw.cuda(), post=Post(-1 / cap, cap, True))
    loss.backward()
    th = torch.tanh(-(h.double() @ w.double().T) / cap)
    want_kl, dkl = odist.divergence(cap * th, ids, t)
    assert (kl.cpu().double() - want_kl).abs().max() <= 1e-4
    dz = dkl * rw.double()[:, None] * -(1 - th ** 2)
    for got, want in [(wd.grad, dz.T @ h.double()), (hd.grad, dz @ w.double())]:
        once = (want.to(torch.bfloat16).double() - want).norm()
        assert (got.cpu().double() - want).norm() <= 2.5 ** 0.5 * once
