"""checkpoint8 and held8 without a GPU: on CPU tensors they are the ordinary checkpoint, with its checks."""

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


# ---- held8 and other checkpoints, with stand-ins for the kernels -----------------------------------------------------

@pytest.fixture
def held(monkeypatch):
    """Rows in 8 bits on the CPU; the widths that were held."""
    calls = []

    def quantise(x, group):
        calls.append(group)
        scale = x.detach().abs().amax(-1, keepdim=True) / 127
        return (x.detach() / scale).round().to(torch.int8), scale

    monkeypatch.setattr(int8_op, "_holds", lambda x, *a: isinstance(x, torch.Tensor) and x.requires_grad and
                        torch.is_grad_enabled() and not isinstance(x, torch.nn.Parameter))
    monkeypatch.setattr(int8_op, "quantise_rows", quantise)
    monkeypatch.setattr(int8_op, "widen_rows", lambda q, s, dtype, group: (q * s).to(dtype))
    return calls


def _grads(y, *of):
    return torch.autograd.grad(y.sum(), of)


@pytest.mark.parametrize("inside", [True, False])
def test_held8_around_another_checkpoint(held, inside):
    """Tiles of a function that a checkpoint recomputes are as without held8(), whether or not it is still open then."""
    x = torch.randn(1, 6, 8, requires_grad=True)
    outer = lambda t: _plain(lambda u: seq_tiles.tiled(torch.sin, u * 2), t)  # noqa: E731
    want = _grads(outer(x), x)
    with seq_tiles.held8(64):
        y = outer(x)
        got = _grads(y, x) if inside else None
    got = got or _grads(y, x)
    assert torch.equal(got[0], want[0]) and not held


def test_held8_inside_another_checkpoint(held):
    """Opened in the function itself it is open in every recompute, and holds 8 bits from each to its backward."""
    def fn(u):
        with seq_tiles.held8(64):
            return seq_tiles.tiled(torch.sin, u * 2)

    x = torch.randn(1, 6, 8, requires_grad=True)
    (got,) = _grads(_plain(fn, x), x)
    q, s = int8_op.quantise_rows(x * 2, 64)
    assert torch.allclose(got, 2 * torch.cos(q * s)) and held == [64] * 3  # the forward, the recompute, this test
    held.clear()
    with seq_tiles.held8(32):
        y = seq_tiles.tiled(torch.sin, x)
    assert torch.allclose(_grads(y, x)[0], torch.cos(int8_op.widen_rows(*int8_op.quantise_rows(x, 32), x.dtype, 32)))


def test_held8_tiles_inside_tiles(held):
    x = torch.randn(1, 6, 8, requires_grad=True)
    with seq_tiles.held8(64):
        y = seq_tiles.tiled(lambda t: seq_tiles.tiled(torch.sin, t) * 2, x)
    assert held == [64]
    _grads(y, x)
    assert held == [64]


def test_held8_and_an_offload(held):
    """Hooks of saved tensors set inside held8() see the tensors as they are, those around it the 8 bits."""
    x = torch.randn(1, 6, 8, requires_grad=True)
    seen = []
    pack = lambda t: seen.append(t.dtype) or t  # noqa: E731
    hooks = lambda: torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t)  # noqa: E731
    with seq_tiles.held8(), hooks():
        y = seq_tiles.tiled(torch.sin, x)
    assert not held and torch.int8 not in seen
    assert torch.equal(_grads(y, x)[0], torch.cos(x.detach()))
    with hooks(), seq_tiles.held8():
        seq_tiles.tiled(torch.sin, x)
    assert held == [128] and torch.int8 in seen
