"""checkpoint8 on the GPU where the recompute could differ from the forward by more than the 8 bits: random numbers,
hooks of saved tensors, tensors that 8 bits do not make smaller."""

import pytest
import torch

from octopus_amd import int8_op

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_random_numbers_are_those_of_the_forward():
    """Dropout in fn, every tensor argument held: the recompute draws the forward's mask, and leaves the generator where
    it was."""
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [0, 128])
def test_rows_that_8_bits_do_not_make_smaller_are_kept(dtype, group, monkeypatch):
    """Rows are padded to 16 bytes and have a scale: a narrow tensor takes fewer bytes as it is."""
    calls = []
    real = int8_op.quantise_rows
    monkeypatch.setattr(int8_op, "quantise_rows", lambda x, g: calls.append(x.shape[-1]) or real(x, g))
    size = torch.finfo(dtype).bits // 8
    for d in (1, 2, 5, 8, 9, 10, 11, 12, 16, 17, 18, 19, 40, 200):
        x = torch.randn(7, d, device=DEV).to(dtype).requires_grad_(True)
        calls.clear()
        (grad,) = torch.autograd.grad(int8_op.checkpoint8(torch.sin, x, group=group).sum(), x)
        smaller = -(-d // 16) * 16 + 4 * (-(-d // group) if group else 1) < d * size
        assert calls == ([d] if smaller else [])
        if not smaller:
            assert torch.equal(grad, torch.cos(x.detach()))


def test_expanded_tensors_are_kept(monkeypatch):
    calls = []
    real = int8_op.quantise_rows
    monkeypatch.setattr(int8_op, "quantise_rows", lambda x, g: calls.append(x.shape) or real(x, g))
    bias = torch.randn(1, 4, 64, device=DEV).requires_grad_(True)
    x = torch.randn(8, 4, 64, device=DEV).requires_grad_(True)
    y = int8_op.checkpoint8(lambda a, b: torch.sin(a + b), x, bias.expand(8, 4, 64))
    gx, gb = torch.autograd.grad(y.sum(), (x, bias))
    assert calls == [(8, 4, 64)] and torch.allclose(gx.sum(0, keepdim=True), gb, rtol=0, atol=8 * 2.0 ** -22)


class _Marked(torch.Tensor):
    """A tensor that fn tells from a plain one."""


def test_subclasses_are_kept():
    x = torch.randn(9, 64, device=DEV).as_subclass(_Marked).requires_grad_(True)
    fn = lambda t: torch.sin(t * (2.0 if isinstance(t, _Marked) else 3.0))  # noqa: E731
    (got,) = torch.autograd.grad(int8_op.checkpoint8(fn, x).sum(), x)
    assert torch.equal(got, 2 * torch.cos(2 * x.detach()))


def test_captured():
    """Both passes in one graph, replayed on new values between the program's own passes."""
    w = torch.randn(256, 200, device=DEV).requires_grad_(True)
    static = torch.randn(33, 256, device=DEV).requires_grad_(True)

    def step(x):
        y = int8_op.checkpoint8(lambda t: torch.sin(t @ w), x)
        return (y.detach(), *torch.autograd.grad(y.sum(), (x, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    for seed in (1, 2, 3):
        new = torch.randn(33, 256, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).requires_grad_(True)
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(new)))
