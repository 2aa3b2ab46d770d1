"""Rows held in 8 bits (octopus_amd.int8_op) on the GPU: the bytes and scales against exact arithmetic, back again, and
the checkpoint that holds its inputs so."""

import math

import pytest
import torch

from octopus_amd import int8_op
from octopus_amd.rl import seq_tiles
from oracle import rows8 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(n, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    return x.to(dtype)


def _check(x, group):
    q, scale = int8_op.quantise_rows(x.to(DEV), group)
    want_q, want_s = oracle.quantise(x.reshape(-1, x.shape[-1]), group)
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.dtype == torch.float32
    assert torch.equal(q.cpu().reshape(want_q.shape).long(), want_q)
    torch.testing.assert_close(scale.cpu().reshape(want_s.shape).double(), want_s, rtol=0, atol=0, equal_nan=True)
    for dtype in TYPES:
        back = int8_op.widen_rows(q, scale, dtype, group)
        want = oracle.widen(want_q, want_s, group).reshape(x.shape)
        assert back.dtype == dtype and back.shape == x.shape
        # a product of 7 by 24 bits, rounded to fp32 and then on
        torch.testing.assert_close(back.cpu(), want.float().to(dtype), rtol=0, atol=0, equal_nan=True)
    return q, scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 7, 16, 31, 33, 128, 500, 511, 513, 1027, 4096, 4097, 9001])
def test_rows(d, dtype):
    _check(_rows(5, d, dtype, d), 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("d", [1, 31, 32, 100, 129, 2304, 2303, 4100])
def test_groups(d, group, dtype):
    _check(_rows(6, d, dtype, d + group), group)


def test_exact_quotients():
    """Values whose quotients lie at, and one step of fp32 beside, the halves."""
    for seed, s in enumerate([1.0, 0.75, 1.0 / 3.0, 3e-30, 7e20]):
        scale = float(torch.tensor(s))
        g = torch.Generator().manual_seed(seed)
        k = torch.randint(-126, 126, (1, 2000), generator=g).double() + 0.5
        x = (k * scale).float()
        near = torch.randint(-2, 3, x.shape, generator=g)
        x = (x.view(torch.int32) + near.int()).view(torch.float32)
        x[0, 0] = 127 * scale
        q, got = int8_op.quantise_rows(x.to(DEV))
        want_q, want_s = oracle.quantise(x, exact=True)
        assert torch.equal(q.cpu().long(), want_q) and got.item() == want_s.item()


def test_rows_without_a_scale():
    x = torch.zeros(6, 70)
    x[1] = 2.0 ** -120                       # below what is held
    x[2, 5] = 2.0 ** -119                    # the least that is
    x[3, 3] = math.nan
    x[4, 69] = -math.inf
    x[5, 1] = -3.0e38
    for group in (0, 32):
        q, scale = _check(x, group)
        back = int8_op.widen_rows(q, scale, torch.float32, group).cpu()
        assert (back[0] == 0).all() and (back[1] == 0).all() and back[2, 5] == 2.0 ** -119
        assert torch.isnan(back[3, :32]).all() and torch.isnan(back[4, 64:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dtype):
    wide = _rows(40, 203, dtype)
    for x in (wide[:, 1:100], wide[::2, 3:], wide.t(), wide[:0], wide[3], wide.reshape(4, 10, 203)[:, :, :64],
              wide[:1].expand(7, 203)):
        for group in (0, 64):
            _check(x, group)


def test_bytes_behind_the_rows():
    x = _rows(9, 37, torch.bfloat16)
    q, _ = int8_op.quantise_rows(x.to(DEV))
    assert q.stride() == (48, 1)
    assert (q.as_strided((9, 48), (48, 1))[:, 37:] == 0).all()
    loose = q.cpu().contiguous().to(DEV)  # rows off their boundaries are copied
    assert torch.equal(int8_op.widen_rows(loose, torch.ones(9, device=DEV), torch.float32).cpu(), q.cpu().float())


def test_refusals():
    x = _rows(4, 64, torch.bfloat16).to(DEV)
    q, scale = int8_op.quantise_rows(x)
    for call in (lambda: int8_op.quantise_rows(x, 48), lambda: int8_op.widen_rows(q, scale, torch.bfloat16, 32),
                 lambda: int8_op.widen_rows(q.to(torch.int16), scale, torch.bfloat16),
                 lambda: int8_op.widen_rows(q, scale.double(), torch.bfloat16),
                 lambda: int8_op.quantise_rows(x.cpu()), lambda: int8_op.quantise_rows(x[:, :0]),
                 lambda: int8_op.widen_rows(q, scale.cpu(), torch.bfloat16),
                 lambda: int8_op.checkpoint8(lambda a: a, x, group=5)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: int8_op.quantise_rows(x.double()), lambda: int8_op.widen_rows(q, scale, torch.float64)):
        with pytest.raises(NotImplementedError):
            call()


# ---- the checkpoint --------------------------------------------------------------------------------------------------

def _layer(w1, w2):
    def fn(x, mask=None):
        h = torch.nn.functional.silu(x @ w1)
        if mask is not None:
            h = h * mask
        return h @ w2
    return fn


def _loss_grads(run, x, params, c):
    y = run(x)
    grads = torch.autograd.grad((y * c).sum(), (x, *params))
    return y.detach(), grads


@pytest.mark.parametrize("group", [0, 128])
def test_checkpoint8_gradients(group):
    """The forward is fn's own; the gradients are those of fn at what the input's 8 bits stand for."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 33, 200, generator=g).to(DEV).requires_grad_(True)
    w1 = (torch.randn(200, 96, generator=g) / 14).to(DEV).requires_grad_(True)
    w2 = (torch.randn(96, 200, generator=g) / 10).to(DEV).requires_grad_(True)
    c = torch.randn(2, 33, 200, generator=g).to(DEV)
    mask = (torch.rand(2, 33, 1, generator=g) < 0.8).float().to(DEV)
    fn = _layer(w1, w2)
    y, got = _loss_grads(lambda t: int8_op.checkpoint8(fn, t, mask, group=group), x, (w1, w2), c)
    assert torch.equal(y, fn(x, mask).detach())
    q, s = int8_op.quantise_rows(x, group)
    x8 = int8_op.widen_rows(q, s, x.dtype, group).requires_grad_(True)
    _, want = _loss_grads(lambda t: fn(t, mask), x8, (w1, w2), c)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_checkpoint8_keeps_parameters():
    """A parameter among the arguments is there anyway: its gradient is that of its own values."""
    x = torch.randn(9, 64, device=DEV, requires_grad=True)
    w = torch.nn.Parameter(torch.randn(64, 32, device=DEV))
    y = int8_op.checkpoint8(lambda a, b: a @ b, x, w)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert torch.equal(gx, torch.ones_like(y) @ w.detach().t())
    q, s = int8_op.quantise_rows(x, 128)
    assert torch.equal(gw, int8_op.widen_rows(q, s, x.dtype, 128).t() @ torch.ones_like(y))


def test_checkpoint8_twice_and_under_no_grad():
    x = torch.randn(5, 64, device=DEV, requires_grad=True)
    w = torch.randn(64, 64, device=DEV, requires_grad=True)
    with torch.no_grad():
        assert torch.equal(int8_op.checkpoint8(lambda a: a @ w, x), x @ w)
    y = int8_op.checkpoint8(lambda a: torch.sin(a @ w), x)
    one = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    two = torch.autograd.grad(y.sum(), (x, w))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_tiles_hold_8_bits(monkeypatch):
    """seq_tiles.tiled's checkpoints inside held8(), several tiles, an argument that is None; outside it nothing
    changes."""
    monkeypatch.setattr(seq_tiles, "TILE", 16)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, 50, 256, generator=g).to(torch.bfloat16).to(DEV).requires_grad_(True)
    w1 = (torch.randn(256, 64, generator=g) / 16).to(torch.bfloat16).to(DEV).requires_grad_(True)
    w2 = (torch.randn(64, 256, generator=g) / 8).to(torch.bfloat16).to(DEV).requires_grad_(True)
    c = torch.randn(1, 50, 256, generator=g).to(torch.bfloat16).to(DEV)
    fn = _layer(w1, w2)
    plain, grads = _loss_grads(lambda t: seq_tiles.tiled(fn, t, None), x, (w1, w2), c)
    calls = []
    real = int8_op.quantise_rows
    monkeypatch.setattr(int8_op, "quantise_rows", lambda *a: calls.append(a[1]) or real(*a))
    with seq_tiles.held8():
        y, got = _loss_grads(lambda t: seq_tiles.tiled(fn, t, None), x, (w1, w2), c)
    assert calls == [128] * 4 and torch.equal(y, plain)
    q, s = real(x, 128)
    x8 = int8_op.widen_rows(q, s, x.dtype, 128).requires_grad_(True)
    _, want = _loss_grads(lambda t: seq_tiles.tiled(fn, t, None), x8, (w1, w2), c)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(calls) == 4
    with seq_tiles.held8(), seq_tiles.no_inner():
        _, inner = _loss_grads(lambda t: seq_tiles.tiled(fn, t, None), x, (w1, w2), c)
    assert len(calls) == 4 and all(torch.equal(a, b) for a, b in zip(inner, grads))
    with pytest.raises(ValueError):
        with seq_tiles.held8(100):
            pass
