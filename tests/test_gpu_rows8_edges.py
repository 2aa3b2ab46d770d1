"""Quotients of the smallest rows that are held (octopus_amd.int8_op.quantise_rows), where half a scale is no number of
fp32."""

import pytest
import torch

from octopus_amd import int8_op
from oracle import rows8 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("group", [0, 32])
def test_quotients_of_the_lowest_binades(group):
    """Values at, and a step of fp32 beside, the halves of scales below 2^-124, odd in their last place."""
    g = torch.Generator().manual_seed(1)
    rows = []
    for e in (-119, -118, -117):
        top = torch.ldexp(1 + torch.randint(0, 1 << 23, (40, 1), generator=g).double() * 2.0 ** -23, torch.tensor(e))
        scale = (top.float() * (torch.tensor(1.0) / torch.tensor(127.0))).double()
        k = torch.randint(-126, 126, (40, 512), generator=g).double() + 0.5
        steps = torch.randint(-2, 3, (40, 512), generator=g).double()
        x = ((k * scale) * 2.0 ** 149).round() + steps  # whole multiples of the least step of fp32
        x = (x * 2.0 ** -149).float()
        x[:, ::32] = top.float()
        rows.append(x)
    x = torch.cat(rows)
    q, s = int8_op.quantise_rows(x.to(DEV), group)
    want_q, want_s = oracle.quantise(x, group, exact=True)
    assert torch.equal(s.cpu().double().reshape(want_s.shape), want_s)
    assert torch.equal(q.cpu().long(), want_q)
