"""int8_head and its gradients where the first tests did not go: saved rows that a hook gives back in another layout,
tangents of forward mode."""

import pytest
import torch

from octopus_amd import int8_op
from tests.test_gpu_int8_head import _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("n", [1, 2, 70, 200])
def test_saved_rows_in_another_layout(n):
    """A hook that gives the 8-bit rows back without the bytes between them: the same gradients."""
    x, w = _inputs(n, 45, 300, torch.bfloat16)
    up = (torch.randn(n, 300, generator=torch.Generator().manual_seed(1)) / 8).bfloat16().to(DEV)
    h, p = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    wq, ws = int8_op.quantise_rows(p)
    want = torch.autograd.grad(int8_op.int8_head(h, wq, ws, weight=p), (h, p), up)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        z = int8_op.int8_head(h, wq, ws, weight=p)
    got = torch.autograd.grad(z, (h, p), up)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_tangents_are_refused():
    """Forward mode has no derivative here: an error, not logits without their tangent."""
    import torch.autograd.forward_ad as fwad

    x, w = _inputs(6, 32, 50, torch.float32)
    x, w = x.to(DEV), w.to(DEV)
    wq, ws = int8_op.quantise_rows(w)
    for grad in (False, True):
        with fwad.dual_level():
            dual = fwad.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
            with pytest.raises((RuntimeError, NotImplementedError)):
                int8_op.int8_head(dual, wq, ws)
            with pytest.raises((RuntimeError, NotImplementedError)):
                int8_op.int8_head(x, wq, ws, weight=fwad.make_dual(w.clone(), torch.ones_like(w)))
    with fwad.dual_level():
        plain = int8_op.int8_head(x, wq, ws)  # no tangent: as ever
    assert torch.equal(plain, int8_op.int8_head(x, wq, ws))
