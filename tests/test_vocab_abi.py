"""The C ABI of the lists and the embedding without a GPU: every refusal comes back before anything is queued."""

import ctypes

import pytest

from octopus_amd import _lib

P = ctypes.c_void_p(4096)  # never read: the calls end at their checks


def _refused(name, *args, exc=ValueError):
    with pytest.raises(exc):
        _lib.call(name, *args)


def test_topk_checks():
    ok = dict(z=P, ld=100, dt=_lib.BF16, n=4, V=100, inv_T=1.0, k=5, ids=P, logp=P, ws=None, nws=0)
    for change in [dict(ld=99), dict(V=0), dict(n=-1), dict(n=1 << 31), dict(dt=_lib.FP8E4M3), dict(inv_T=0.0),
                   dict(inv_T=float("nan")), dict(k=0), dict(k=101), dict(V=1000, ld=1000, k=257), dict(z=None),
                   dict(ids=None), dict(logp=None), dict(z=ctypes.c_void_p(4097))]:
        _refused("octo_topk", *{**ok, **change}.values(), None)
    _lib.call("octo_topk", *{**ok, "n": 0}.values(), None)
    out = ctypes.c_size_t(0)
    _lib.call("octo_topk_workspace_bytes", 2048, 151936, _lib.BF16, 64, ctypes.byref(out))
    assert out.value == 0
    _lib.call("octo_topk_workspace_bytes", 3, 151936, _lib.BF16, 64, ctypes.byref(out))
    assert out.value > 0
    few = {**ok, "n": 3, "V": 151936, "ld": 151936, "k": 64}
    for change in [dict(), dict(ws=P, nws=out.value - 1), dict(ws=ctypes.c_void_p(4100), nws=out.value)]:
        _refused("octo_topk", *{**few, **change}.values(), None)
    for n, V, k in [(-1, 100, 5), (4, 0, 5), (4, 100, 0), (4, 100, 101), (4, 1000, 257)]:
        _refused("octo_topk_workspace_bytes", n, V, _lib.F32, k, ctypes.byref(out))
    _refused("octo_topk_workspace_bytes", 4, 100, _lib.F16, 5, None)
    _refused("octo_topk_workspace_bytes", 4, 100, _lib.FP8E4M3, 5, ctypes.byref(out))


def test_distill_columns_checks():
    ok = dict(z=P, ld=100, dt=_lib.F16, ids=P, t=P, n=4, V=100, K=5, inv_T=1.0, flags=0, kl=P, state=P, q=P)
    for change in [dict(ld=99), dict(V=0), dict(n=-1), dict(n=1 << 31), dict(dt=_lib.FP8E4M3), dict(dt=-1),
                   dict(inv_T=-1.0), dict(K=0), dict(K=257), dict(flags=2), dict(z=None), dict(ids=None), dict(t=None),
                   dict(kl=None), dict(state=None), dict(q=None), dict(z=ctypes.c_void_p(4097))]:
        _refused("octo_distill_columns_fwd", *{**ok, **change}.values(), None)
    _lib.call("octo_distill_columns_fwd", *{**ok, "n": 0}.values(), None)
    ok = dict(z=P, ld=100, dt=_lib.F32, ids=P, q=P, n=4, V=100, K=5, inv_T=1.0, state=P, g=P, dz=P, ld_d=100)
    for change in [dict(ld=99), dict(ld_d=99), dict(V=0), dict(n=-1), dict(dt=_lib.FP8E4M3), dict(inv_T=0.0), dict(K=0),
                   dict(K=257), dict(z=None), dict(ids=None), dict(q=None), dict(state=None), dict(g=None),
                   dict(dz=None), dict(dz=ctypes.c_void_p(4098))]:
        _refused("octo_distill_columns_bwd", *{**ok, **change}.values(), None)
    _lib.call("octo_distill_columns_bwd", *{**ok, "n": 0}.values(), None)


def test_embed_checks():
    ok = dict(w=P, ldw=64, dt=_lib.BF16, V=10, d=64, ids=P, n=4, scale=1.0, out=P, ldo=64)
    for change in [dict(ldw=63), dict(ldo=63), dict(V=0), dict(d=0), dict(n=-1), dict(n=1 << 31), dict(V=1 << 31),
                   dict(w=None), dict(ids=None), dict(out=None), dict(w=ctypes.c_void_p(4097))]:
        _refused("octo_embed_fwd", *{**ok, **change}.values(), None)
    _refused("octo_embed_fwd", *{**ok, "dt": _lib.FP8E4M3}.values(), None, exc=NotImplementedError)
    _lib.call("octo_embed_fwd", *{**ok, "n": 0}.values(), None)
    out = ctypes.c_size_t(0)
    _lib.call("octo_embed_bwd_workspace_bytes", 4, 10, 64, ctypes.byref(out))
    assert out.value >= 4 * 8 + 11 * 4 + 2 * 64 * 4
    for n, V, d in [(-1, 10, 64), ((1 << 30) + 1, 10, 64), (4, 0, 64), (4, 1 << 31, 64), (4, 10, 0), (4, 10, 1 << 30)]:
        _refused("octo_embed_bwd_workspace_bytes", n, V, d, ctypes.byref(out))
    _refused("octo_embed_bwd_workspace_bytes", 4, 10, 64, None)
    _lib.call("octo_embed_bwd_workspace_bytes", 4, 10, 64, ctypes.byref(out))
    ok = dict(g=P, ldg=64, gdt=_lib.BF16, ids=P, n=4, V=10, d=64, pad=-1, scale=1.0, gw=P, ldw=64, wdt=_lib.BF16, acc=0,
              ws=P, nws=out.value)
    for change in [dict(ldg=63), dict(ldw=63), dict(n=-1), dict(V=0), dict(d=0), dict(g=None), dict(ids=None),
                   dict(gw=None), dict(ws=None), dict(nws=out.value - 1), dict(gw=ctypes.c_void_p(4097)),
                   dict(ws=ctypes.c_void_p(4104))]:
        _refused("octo_embed_bwd", *{**ok, **change}.values(), None)
    for change in [dict(gdt=_lib.FP8E4M3), dict(wdt=7)]:
        _refused("octo_embed_bwd", *{**ok, **change}.values(), None, exc=NotImplementedError)


def test_python_checks_need_no_gpu():
    """Shapes, sizes and devices are refused before a tensor is read; a CPU tensor has no kernel."""
    import torch

    from octopus_amd import distill_op, embed_op

    z, ids, t = torch.zeros(3, 50), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4)
    for call in [lambda: distill_op.head_topk(z, 1.0, 0), lambda: distill_op.head_topk(z, 1.0, 51),
                 lambda: distill_op.head_topk(z, 0.0, 5), lambda: distill_op.head_topk(z[0], 1.0, 5),
                 lambda: distill_op.head_topk(z, 1.0, 5), lambda: distill_op.distill_columns(z[0], 1.0, ids, t),
                 lambda: distill_op.distill_columns(z, -1.0, ids, t), lambda: embed_op.embed_rows(z[0], ids),
                 lambda: embed_op.embed_rows(z, ids), lambda: embed_op.embed_rows(z, ids, padding_idx=3),
                 lambda: distill_op.distill_columns(z, 1.0, ids, t),
                 lambda: embed_op.embed_grad_add_(z[0], t, ids)]:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):  # the registered ops know HIP tensors only
        distill_op.distill_columns_fwd(z, ids, t, 1.0, False)


def test_sizes_past_the_kernels_counts():
    """Vocabularies and token counts whose places, or launches, would not fit 32 bits."""
    V, out = (1 << 30) + 1, ctypes.c_size_t(0)
    _refused("octo_topk", P, V, _lib.BF16, 4, V, 1.0, 5, P, P, None, 0, None)
    _refused("octo_topk_workspace_bytes", 4, V, _lib.BF16, 5, ctypes.byref(out))
    _refused("octo_distill_columns_fwd", P, V, _lib.BF16, P, P, 4, V, 5, 1.0, 0, P, P, P, None)
    _refused("octo_distill_columns_bwd", P, V, _lib.BF16, P, P, 4, V, 5, 1.0, P, P, P, V, None)
    _refused("octo_embed_fwd", P, 8, _lib.BF16, V, 8, P, 4, 1.0, P, 8, None)
    for n, v in [((1 << 27) + 1, 10), (4, V)]:
        _refused("octo_embed_bwd_workspace_bytes", n, v, 8, ctypes.byref(out))


def test_rows_that_go_whole_need_no_workspace():
    """Few fp32 rows from 60,000 values on, and of 16 bits from 192 KB, are cut into slices; shorter ones are faster whole."""
    out = ctypes.c_size_t(0)
    for n, V, dtype, k, sliced in [(1, 49152, _lib.F32, 64, False), (1, 59999, _lib.F32, 64, False),
                                   (1, 60000, _lib.F32, 64, True), (128, 98304, _lib.BF16, 128, True),
                                   (128, 98303, _lib.F16, 128, False), (129, 151936, _lib.BF16, 64, False),
                                   (1, 151936, _lib.BF16, 129, False)]:
        _lib.call("octo_topk_workspace_bytes", n, V, dtype, k, ctypes.byref(out))
        assert (out.value > 0) == sliced
