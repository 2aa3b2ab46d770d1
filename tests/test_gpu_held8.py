"""checkpoint8 on the GPU where the recompute could differ from the forward by more than the 8 bits: random numbers, hooks
of saved tensors, tensors that 8 bits do not make smaller."""

import pytest
import torch

from octopus_amd import int8_op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_random_numbers_are_those_of_the_forward():
    """Dropout in fn, every tensor argument held: the recompute draws the forward's mask, and leaves the generator where it
    was."""
    x = torch.randn(64, 256, device=DEV).requires_grad_(True)
    y = int8_op.checkpoint8(lambda t: torch.nn.functional.dropout(t, 0.5).square(), x)
    torch.rand(3, device=DEV)
    state = torch.cuda.get_rng_state()
    (grad,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(torch.cuda.get_rng_state(), state)
    # the gradient is 2 x mask^2 of the x that the 8 bits stand for: zero where they are zero, or the forward's mask is
    assert torch.equal(grad == 0, (y == 0) | (int8_op.quantise_rows(x, 128)[0] == 0))


def test_held_rows_through_hooks_of_saved_tensors():
    """An offload's hooks see the 8 bits and their scales, and may give them back in another layout."""
    x = torch.randn(9, 203, device=DEV).requires_grad_(True)
    want = torch.autograd.grad(int8_op.checkpoint8(torch.sin, x).sum(), x)
    packed = []

    def pack(t):
        if t.numel():
            packed.append((t.dtype, t.numel()))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        y = int8_op.checkpoint8(torch.sin, x)
    got = torch.autograd.grad(y.sum(), x)
    assert torch.equal(got[0], want[0])
    assert packed == [(torch.int8, 9 * 203), (torch.float32, 9 * 2)]


def test_held8_around_another_checkpoint():
    """The tiles of a layer that a checkpoint recomputes, with the backward behind held8(): as without it."""
    from torch.utils.checkpoint import checkpoint

    from octopus_amd.rl import seq_tiles

    x = torch.randn(1, 50, 256, device=DEV).requires_grad_(True)
    layer = lambda t: checkpoint(lambda u: seq_tiles.tiled(torch.sin, u * 2), t, use_reentrant=False)  # noqa: E731
    (want,) = torch.autograd.grad(layer(x).sum(), x)
    with seq_tiles.held8():
        y = layer(x)
    (got,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(got, want)
