"""checkpoint8 and held8 where nothing is held in 8 bits: on CPU tensors they are the ordinary checkpoint, with its checks."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from octopus_amd import int8_op
from octopus_amd.rl import seq_tiles


def _plain(fn, *xs):
    return checkpoint(fn, *xs, use_reentrant=False)


def _tiled(fn, *xs):
    with seq_tiles.held8():
        return seq_tiles.tiled(fn, *xs)


@pytest.mark.parametrize("run", [_plain, int8_op.checkpoint8, _tiled])
@pytest.mark.parametrize("what", ["mask", "parameter", "input"])
def test_arguments_changed_in_place_are_refused(run, what):
    """What the recompute would read again, changed between the passes: an error, not another gradient."""
    x = torch.randn(1, 6, 8).requires_grad_(True)
    mask = torch.ones(1, 6, 8)
    w = torch.nn.Parameter(torch.randn(1, 6, 8))
    inner = x * 1
    y = run(lambda a, m, p: torch.sin(a * m * p), inner, mask, w)
    with torch.no_grad():
        {"mask": mask.zero_, "parameter": lambda: w.mul_(1.5), "input": lambda: inner.mul_(2)}[what]()
    with pytest.raises(RuntimeError, match="modified (by an )?inplace"):
        torch.autograd.grad(y.sum(), (x, w))


@pytest.mark.parametrize("run", [_plain, int8_op.checkpoint8, _tiled])
def test_arguments_pass_as_they_are(run):
    x, w = torch.randn(1, 6, 8, requires_grad=True), torch.randn(1, 6, 8, requires_grad=True)
    fn = lambda a, none, b: torch.sin(a * b) if none is None else a  # noqa: E731
    got = torch.autograd.grad(run(fn, x, None, w).sum(), (x, w))
    want = torch.autograd.grad(fn(x, None, w).sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
