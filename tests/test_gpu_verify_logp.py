"""The log-probabilities of verify_drafts on both routes: within one rounding of their value where the rows' sums are
taken in 64 bits (few logits, and every drawn token), within 5e-6 and one rounding where they are of 32-bit exponentials
(2^24 logits and more: the accepted drafts, and greedy's tokens)."""

import pytest
import torch

from octopus_amd import verify_op
from oracle import verify as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _logits(S, K, V, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = torch.randn(S, K + 1, V, generator=g, device=DEV) * 2.5
    best = torch.randint(0, V, (S, K + 1, 1), generator=g, device=DEV)
    z.scatter_(2, best, 14.0)  # one likely token a row, so that drafts of it are accepted
    return z.to(dtype), best[:, :K, 0].clone(), torch.rand(S, K + 1, generator=g, device=DEV)


def _rounded(lp):
    return 2.0 ** -24 * lp.abs() + 1e-12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("greedy", [True, False])
def test_many_logits(dtype, greedy):
    S, K, V = 62, 2, 100003  # 18.6M logits
    z, x, u = _logits(S, K, V, dtype, 1)
    x[::5, 1] = (x[::5, 1] + 1) % V
    tokens, accepted, logp = verify_op.verify_drafts(z, x, u, 0.9, greedy=greedy)
    lp = torch.log_softmax(z.double() / 0.9, 2)
    assert 0 < accepted.sum() < S * K
    want = lp.gather(2, tokens.clamp(min=0)[:, :, None])[:, :, 0] * (tokens >= 0)
    at = torch.arange(K + 1, device=DEV)[None]
    exact = (at >= accepted[:, None]) & (not greedy)  # the drawn token, and the zeros behind it
    bound = _rounded(want) + torch.where(exact, 0.0, 5e-6)
    assert ((logp.double() - want).abs() <= bound).all()
    # a sequence by itself: the same tokens, its log-probabilities within one rounding
    for s in (0, 1, 33):
        alone = verify_op.verify_drafts(z[s:s + 1], x[s:s + 1], u[s:s + 1], 0.9, greedy=greedy)
        assert torch.equal(alone[0][0], tokens[s]) and alone[1][0] == accepted[s]
        assert ((alone[2][0].double() - want[s]).abs() <= _rounded(want[s])).all()
    if greedy:
        one = oracle.verify(z[:1].cpu(), x[:1].cpu(), None, 0.9, greedy=True)
        assert one[0][0] == tokens[0].tolist()
