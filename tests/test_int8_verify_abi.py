"""The C ABI of the 8-bit rows, the 8-bit head and the verification without a GPU: every refusal comes back before
anything is queued. Their oracles pinned, and the checkpoint's refusals."""

import ctypes
import math

import pytest
import torch

from octopus_amd import _lib, int8_op
from oracle import rows8, verify

P = ctypes.c_void_p(4096)  # never read: the calls end at their checks


def _refused(name, *args, exc=ValueError):
    with pytest.raises(exc):
        _lib.call(name, *args)


def test_rows8_checks():
    ok = dict(x=P, ldx=64, dt=_lib.BF16, rows=4, d=60, group=0, q=P, ldq=64, scale=P)
    for change in [dict(ldx=59), dict(rows=-1), dict(rows=1 << 31), dict(d=0), dict(group=16), dict(group=100),
                   dict(group=512), dict(ldq=60), dict(ldq=48), dict(x=None), dict(q=None), dict(scale=None),
                   dict(x=ctypes.c_void_p(4097)), dict(q=ctypes.c_void_p(4104)), dict(scale=ctypes.c_void_p(4098))]:
        _refused("octo_quantise_i8_rows", *{**ok, **change}.values(), None)
    _refused("octo_quantise_i8_rows", *{**ok, "dt": _lib.FP8E4M3}.values(), None, exc=NotImplementedError)
    _lib.call("octo_quantise_i8_rows", *{**ok, "rows": 0}.values(), None)
    ok = dict(q=P, ldq=64, scale=P, rows=4, d=60, group=32, out=P, ldo=60, dt=_lib.F32)
    for change in [dict(ldo=59), dict(rows=-1), dict(d=0), dict(group=33), dict(ldq=56), dict(q=None), dict(scale=None),
                   dict(out=None), dict(out=ctypes.c_void_p(4098)), dict(q=ctypes.c_void_p(4097))]:
        _refused("octo_widen_i8_rows", *{**ok, **change}.values(), None)
    _refused("octo_widen_i8_rows", *{**ok, "dt": 7}.values(), None, exc=NotImplementedError)
    _lib.call("octo_widen_i8_rows", *{**ok, "rows": 0}.values(), None)


def test_head8_checks():
    ok = dict(x=P, ldx=60, xdt=_lib.BF16, wq=P, ldw=64, ws=P, n=4, d=60, V=100, xq=P, ldxq=64, xs=P, z=P, ldz=100,
              zdt=_lib.F16)
    for change in [dict(ldx=59), dict(ldw=60), dict(ldw=48), dict(n=-1), dict(n=(1 << 21) + 1), dict(d=0),
                   dict(d=131073, ldx=131073, ldw=131088, ldxq=131088), dict(V=0), dict(V=(1 << 21) + 1, ldz=1 << 22),
                   dict(ldxq=63), dict(ldz=99), dict(wq=None), dict(ws=None), dict(xq=None), dict(xs=None),
                   dict(z=None), dict(wq=ctypes.c_void_p(4104)), dict(z=ctypes.c_void_p(4097)),
                   dict(x=ctypes.c_void_p(4097))]:
        _refused("octo_head_logits_i8", *{**ok, **change}.values(), None)
    for change in [dict(zdt=_lib.FP8E4M3), dict(xdt=_lib.FP8E4M3)]:
        _refused("octo_head_logits_i8", *{**ok, **change}.values(), None, exc=NotImplementedError)
    _lib.call("octo_head_logits_i8", *{**ok, "n": 0}.values(), None)
    out = ctypes.c_size_t(0)
    for n, d, V in [(-1, 60, 100), (4, 0, 100), (4, 60, 0), (4, 131073, 100), (4, 60, (1 << 21) + 1)]:
        _refused("octo_head_grads_i8_workspace_bytes", P, V, _lib.BF16, n, d, V, 1, 1, ctypes.byref(out))
    _refused("octo_head_grads_i8_workspace_bytes", P, 100, _lib.BF16, 4, 60, 100, 1, 1, None)
    # a gradient that is read where it lies needs no copy
    size = lambda p, ld, dt, V: _lib.call("octo_head_grads_i8_workspace_bytes", p, ld, dt, 640, 64, V, 0, 1,  # noqa: E731
                                          ctypes.byref(out)) or out.value
    copy = 640 * 1024 * 2
    assert size(P, 1000, _lib.BF16, 1000) + copy == size(P, 1001, _lib.BF16, 1000)
    assert size(P, 1001, _lib.BF16, 1000) == size(ctypes.c_void_p(4098), 1000, _lib.BF16, 1000) \
        == size(P, 1008, _lib.BF16, 999)
    _lib.call("octo_head_grads_i8_workspace_bytes", P, 100, _lib.BF16, 4, 60, 100, 1, 1, ctypes.byref(out))
    ok = dict(g=P, ldg=100, gdt=_lib.BF16, xq=P, ldxq=64, xs=P, wq=P, ldw=64, ws=P, n=4, d=60, V=100, gr=P, ldr=60,
              rdt=_lib.BF16, gw=P, ldgw=60, wdt=_lib.BF16, work=P, nwork=out.value)
    for change in [dict(ldg=99), dict(ldr=59), dict(ldgw=59), dict(n=0), dict(n=-1), dict(d=0), dict(V=0), dict(g=None),
                   dict(xq=None), dict(xs=None), dict(wq=None), dict(ws=None), dict(work=None),
                   dict(nwork=out.value - 1), dict(work=ctypes.c_void_p(4112)), dict(ldxq=60), dict(ldw=32),
                   dict(g=ctypes.c_void_p(4097)), dict(gw=ctypes.c_void_p(4097))]:
        _refused("octo_head_grads_i8", *{**ok, **change}.values(), None)
    _refused("octo_head_grads_i8", *{**ok, "gdt": 9}.values(), None, exc=NotImplementedError)
    far = dict(gdt=_lib.F32, nwork=1 << 62)  # three parts of fp32 gradients lie within 32-bit offsets up to 2^20
    _refused("octo_head_grads_i8", *{**ok, **far, "n": (1 << 20) + 1}.values(), None)
    _refused("octo_head_grads_i8", *{**ok, **far, "V": (1 << 20) + 1, "ldg": 1 << 21}.values(), None)
    _lib.call("octo_head_grads_i8", *{**ok, "gr": None, "gw": None}.values(), None)


def test_verify_checks():
    out = ctypes.c_size_t(0)
    for S, K, V in [(-1, 4, 100), ((1 << 20) + 1, 4, 100), (4, -1, 100), (4, 64, 100), (4, 4, 0), (4, 4, (1 << 30) + 1)]:
        _refused("octo_verify_workspace_bytes", S, K, V, ctypes.byref(out))
    _refused("octo_verify_workspace_bytes", 4, 4, 100, None)
    _lib.call("octo_verify_workspace_bytes", 4, 3, 100, ctypes.byref(out))
    ok = dict(z=P, ls=400, lr=100, zd=P, lsd=300, lrd=100, dt=_lib.BF16, x=P, n=None, u=P, S=4, K=3, V=100, it=1.0,
              greedy=0, tokens=P, acc=P, logp=P, ws=P, nws=out.value)
    for change in [dict(ls=-1), dict(lr=-1), dict(lsd=-1), dict(z=None), dict(x=None), dict(u=None), dict(tokens=None),
                   dict(acc=None), dict(logp=None), dict(ws=None), dict(nws=out.value - 1), dict(it=0.0),
                   dict(it=math.nan), dict(it=1e39), dict(S=-1), dict(K=64), dict(V=0), dict(z=ctypes.c_void_p(4097)),
                   dict(zd=ctypes.c_void_p(4097)), dict(ws=ctypes.c_void_p(4104))]:
        _refused("octo_verify_drafts", *{**ok, **change}.values(), None)
    _refused("octo_verify_drafts", *{**ok, "dt": _lib.FP8E4M3}.values(), None, exc=NotImplementedError)
    _lib.call("octo_verify_drafts", *{**ok, "S": 0}.values(), None)


def test_cpu_tensors_are_refused():
    x = torch.ones(2, 32)
    with pytest.raises(ValueError):
        int8_op.quantise_rows(x)
    with pytest.raises(ValueError):
        int8_op.quantise_rows(x, 7)


def test_fp32_gradients_too_large_are_refused_before_the_forward():
    big = (1 << 20) + 1
    wq, ws = torch.zeros(1, 4, dtype=torch.int8).expand(big, 4), torch.ones(1).expand(big)
    for x, q, s in ((torch.zeros(1, 4), wq, ws), (torch.zeros(1, 4).expand(big, 4), wq[:3], ws[:3])):
        with pytest.raises(ValueError, match="fp32 logits"):
            int8_op.int8_head(x.detach().requires_grad_(True), q, s)


def test_checkpoint8_keeps_cpu_tensors():
    """CPU tensors are checkpointed as they are, so the seq tiles' CPU tests read the same inside held8()."""
    from octopus_amd.rl import seq_tiles
    x, w = torch.randn(1, 9, 8, requires_grad=True), torch.randn(8, 8, requires_grad=True)
    fn = lambda t: torch.tanh(t @ w)  # noqa: E731
    want = torch.autograd.grad(fn(x).square().sum(), (x, w))
    with seq_tiles.held8(0):
        got = torch.autograd.grad(seq_tiles.tiled(fn, x).square().sum(), (x, w))
    assert all(torch.allclose(a, b) for a, b in zip(got, want))
    assert seq_tiles._HELD8 is None
    with pytest.raises(ValueError):
        int8_op.checkpoint8(fn, x, group=3)


def test_oracle_rows8():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, 63.4], [0, 0, 0, 0, 0], [1, -2, 3, -4, 5]])
    q, s = rows8.quantise(x)
    assert q[0].tolist() == [127, 0, 2, -2, 63] and s[:, 0].tolist()[:2] == [1.0, 0.0] and not q[1].any()
    assert q[2].tolist() == [25, -51, 76, -102, 127]
    a, b = rows8.quantise(x, exact=True)
    assert torch.equal(a, q) and torch.equal(b, s)
    q, s = rows8.quantise(torch.randn(4, 10), 4)
    assert s.shape == (4, 3) and rows8.widen(q, s, 4).shape == (4, 10)


@pytest.mark.parametrize("sampled", [True, False])
def test_oracle_verify_answers_with_the_targets_distribution(sampled):
    """Over a fine grid of the random numbers and every draft by its probability, the first token is the target's."""
    z = torch.tensor([[[0.3, -1.0, 1.2, 0.0], [0.0, 0.0, 0.0, 0.0]]])
    zd = torch.tensor([[[1.0, 0.5, -0.7, 0.2]]])
    p, q = torch.softmax(z[0, 0].double(), 0), torch.softmax(zd[0, 0].double(), 0)
    N, got = 60, torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        weight = q[x].item() if sampled else float(x == 1)
        for i in range(N):
            for j in range(N):
                u = torch.tensor([[(i + 0.5) / N, (j + 0.5) / N]])
                t = verify.verify(z, torch.tensor([[x]]), u, 1.0, zd if sampled else None)[0][0][0]
                got[t] += weight / N ** 2
    assert (got - p).abs().max() <= 2.0 / N  # the grid's steps


def test_oracle_verify_greedy_and_masks():
    z = torch.tensor([[[0.0, 2.0, 2.0], [1.0, 0.0, 0.0]], [[-math.inf] * 3, [0.0] * 3]])
    tokens, acc, logp = verify.verify(z, torch.tensor([[1], [0]]), None, 1.0, greedy=True)
    assert tokens == [[1, 0], [-1, -1]] and acc == [1, 0] and math.isnan(logp[1][0])


def test_oracle_verify_dense():
    g = torch.Generator().manual_seed(0)
    z, zd = torch.randn(30, 4, 50, generator=g) * 2, torch.randn(30, 3, 50, generator=g) * 2
    zd[5, :, 9:], z[5, :, 9:] = -math.inf, -math.inf
    x, u = torch.randint(0, 9, (30, 3), generator=g), torch.rand(30, 4, generator=g)
    n = torch.randint(0, 4, (30,), generator=g)
    for d in (zd, None):
        a, b = verify.verify(z, x, u, 0.8, d, n), verify.verify_dense(z, x, u, 0.8, d, n)
        assert a[0] == b[0].tolist() and a[1] == b[1].tolist()
        assert (torch.tensor(a[2], dtype=torch.float64) - b[2]).abs().max() < 1e-12
