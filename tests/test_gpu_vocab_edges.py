"""Calls of the lists, the distillation and the embedding at the edges of what their documentation allows."""

import pytest
import torch

from oracle import distill as odist

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("later", [False, True])
def test_a_soft_cap_of_negative_slope_keeps_the_roundings(later, monkeypatch):
    """z = 30 tanh(-x / 30): the weight gradient of bf16 operands takes two roundings of half a step each, the listed
    values' and the result's, as with a positive slope. Roundings of one size add in squares, so its error lies below
    sqrt(2.5) times the one that the exact gradient's own rounding costs; a third (h^T times a scale that is not a power
    of two) would bring it to sqrt(3)."""
    from octopus_amd import distill_op, head_op
    from octopus_amd.head_op import Post

    n, d, V, K, cap = 300, 256, 8192, 64, 30.0
    g = torch.Generator().manual_seed(21)
    h, w = torch.randn(n, d, generator=g).to(torch.bfloat16), (torch.randn(V, d, generator=g) * 0.02).to(torch.bfloat16)
    ids, t = torch.randint(0, V, (n, K), generator=g), torch.randn(n, K, generator=g)
    rw = torch.rand(n, generator=g) + 0.5
    monkeypatch.setattr(head_op, "_LATER_SHARE", 1 << 20)
    monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 0 if later else 1 << 62)
    monkeypatch.setattr(head_op, "_LATER_WORK", 1 << 62)
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    assert (distill_op._later_bytes(hd, wd, None, True, True) > 0) == later
    loss, kl = distill_op.fused_distill_head(hd, wd, ids.cuda(), t.cuda(), 1.0, rw.cuda(),
                                             post=Post(-1 / cap, cap, True))
    loss.backward()
    th = torch.tanh(-(h.double() @ w.double().T) / cap)
    want_kl, dkl = odist.divergence(cap * th, ids, t)
    assert (kl.cpu().double() - want_kl).abs().max() <= 1e-4
    dz = dkl * rw.double()[:, None] * -(1 - th ** 2)
    for got, want in [(wd.grad, dz.T @ h.double()), (hd.grad, dz @ w.double())]:
        once = (want.to(torch.bfloat16).double() - want).norm()
        assert (got.cpu().double() - want).norm() <= 2.5 ** 0.5 * once


def _small(n=6, d=64, V=300, K=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    w = (torch.randn(V, d, generator=g) * 0.2).to(torch.bfloat16).cuda().requires_grad_(True)
    return h, w, torch.randint(0, V, (n, K), generator=g).cuda(), torch.randn(n, K, generator=g).cuda()


def test_only_one_output_of_the_registered_ops_is_differentiable():
    """A loss of the step's divergences or gradients, or of the divergence's state, raises: a gradient of zeros, or one
    without that part, would be silently wrong."""
    from octopus_amd import distill_op

    h, w, ids, t = _small()
    loss, kl, gh, gw = distill_op.head_step_distill(h, w, None, ids, t, None, None, None, 1.0, 1.0, 1.0, False, False,
                                                    True, True)
    for out in (kl.sum(), gh.float().sum(), gw.float().sum(), loss + kl.sum()):
        with pytest.raises(RuntimeError, match="only loss"):
            torch.autograd.grad(out, (h, w), retain_graph=True)
    a = torch.autograd.grad(loss, (h, w))
    assert torch.equal(a[0], gh) and torch.equal(a[1], gw)
    z = torch.randn(6, 300, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    kl, state, q = distill_op.distill_columns_fwd(z, ids, t, 1.0, False)
    for out in (state.sum(), q.sum(), kl.sum() + q.sum()):
        with pytest.raises(RuntimeError, match="only kl"):
            torch.autograd.grad(out, z, retain_graph=True)
    (a,) = torch.autograd.grad(kl.sum(), z)
    (b,) = torch.autograd.grad(distill_op.distill_columns(z, 1.0, ids, t).sum(), z)
    assert torch.equal(a, b)


def test_traced_steps():
    """Through a tracer: the loss's gradients are the eager call's, the divergences come detached."""
    from octopus_amd import distill_op

    h, w, ids, t = _small(seed=2)

    def step(h, w):
        loss, kl = distill_op.fused_distill_head(h, w, ids, t, 1.0)
        return loss, kl, distill_op.distill_columns((h @ w.T).float(), 1.0, ids, t)

    def all_of(f):
        loss, kl, cols = f(h, w)
        assert not kl.requires_grad
        return (loss.detach(), kl, cols.detach(), *torch.autograd.grad(3 * loss + cols.sum(), (h, w)))

    got = all_of(torch.compile(step, backend="aot_eager", fullgraph=True))
    assert all(torch.equal(a, b) for a, b in zip(got, all_of(step)))


def test_a_traced_lookup_and_its_second_derivative():
    """embed_rows through a tracer has the eager call's gradient; the registered op's gradient, differentiated again,
    raises also as part of a larger expression."""
    from octopus_amd import embed_op

    ids = torch.tensor([[3, 0, 3], [7, -1, 9]], device="cuda")
    w = torch.randn(9, 16, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True)
    up = torch.randn(2, 3, 16, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_(True)
    step = lambda w: embed_op.embed_rows(w, ids, 1.5, padding_idx=7)  # noqa: E731
    out = torch.compile(step, backend="aot_eager", fullgraph=True)(w)
    assert torch.equal(out, step(w))
    (a,) = torch.autograd.grad(out, w, up.detach())
    (b,) = torch.autograd.grad(step(w), w, up.detach())
    assert torch.equal(a, b)
    for f in (embed_op.embed_fwd, lambda *x: embed_op.embed_rows(*x)):
        (g,) = torch.autograd.grad(f(w, ids, 1.5, 7), w, up, create_graph=True)
        assert torch.equal(g, a)
        with pytest.raises(RuntimeError):
            (up.pow(2).sum() + g.pow(2).sum()).backward()


@pytest.mark.parametrize("form", ["step", "later", "registered", "columns", "columns_apart", "registered_columns"])
def test_second_derivatives_inside_a_larger_expression(form, monkeypatch):
    """A penalty on the gradient beside a term that has a derivative: the penalty's own raises by every way that asks
    for it, where a constant in its place would leave it out without a word. The first derivatives are the plain
    ones."""
    from octopus_amd import distill_op, head_op

    h, w, ids, t = _small(seed=5)
    rw = torch.rand(6, generator=torch.Generator().manual_seed(6)).cuda()
    monkeypatch.setattr(head_op, "_LATER_SHARE", 1 << 20)
    monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 0 if form == "later" else 1 << 62)
    monkeypatch.setattr(head_op, "_LATER_WORK", 1 << 62)
    if "columns" in form:
        shape = (300, 6) if form == "columns_apart" else (6, 300)
        x = torch.randn(shape, generator=torch.Generator().manual_seed(7)).cuda()
        x = x.T if form == "columns_apart" else x
        leaves = (x.detach().requires_grad_(True),)
        call = distill_op.distill_columns_fwd if form == "registered_columns" else None
        f = lambda: (call(leaves[0], ids, t, 1.0, False)[0] if call  # noqa: E731
                     else distill_op.distill_columns(leaves[0], 1.0, ids, t)).sum()
    else:
        leaves = (h, w)
        args = (h, w, None, ids, t, rw, None, None, 1.0, 1.0, 1.0, False, False, True, True)
        f = lambda: (distill_op.head_step_distill(*args) if form == "registered"  # noqa: E731
                     else distill_op.fused_distill_head(h, w, ids, t, 1.0, rw))[0]
    want = torch.autograd.grad(f(), leaves)

    def penalised():
        loss = f()
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        return loss + sum(g.float().pow(2).sum() for g in grads) + sum(x.float().sum() for x in leaves)

    with pytest.raises(RuntimeError):
        penalised().backward()
    for x in leaves:
        with pytest.raises(RuntimeError):
            torch.autograd.grad(penalised(), x)


def _fastest(f, calls=10, turns=5):
    """us a call, the fastest of a few runs."""
    for _ in range(3):
        f()
    times = []
    for _ in range(turns):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(calls):
            f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    return min(times)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,d,ld,off", [(1, 1, 1, 0), (1, 3, 9, 5), (3, 1, 1, 1), (5, 7, 7, 3), (37, 41, 41, 0),
                                        (37, 41, 41, 1), (37, 41, 45, 2), (700, 64, 64, 4), (3, 5, 8, 7),
                                        (513, 1031, 1031, 6), (40, 2047, 2050, 1)])
def test_gradients_zeros_end_where_it_does(dtype, V, d, ld, off):
    """The dense gradient at every offset from a 16-byte boundary, of odd lengths, with and without gaps between its
    rows: zeros where no token is, and nothing written around it."""
    import ctypes

    from octopus_amd import _lib
    from octopus_amd.head_op import _DT, _p, _stream

    n = 4
    ids = torch.tensor([V - 1, 0, -1, V - 1], device="cuda")
    g = torch.arange(1, n * d + 1, device="cuda").reshape(n, d).remainder(61).to(dtype)
    base = torch.full((off + V * ld + 40,), 7.0, dtype=dtype, device="cuda")
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_embed_bwd_workspace_bytes", n, V, d, ctypes.byref(nbytes))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device="cuda")
    inner = base[off:off + V * ld].view(V, ld)[:, :d]
    _lib.call("octo_embed_bwd", _p(g), d, _DT[dtype], _p(ids), n, V, d, -1, 1.0, ctypes.c_void_p(inner.data_ptr()), ld,
              _DT[dtype], 0, _p(ws), ws.numel(), _stream(g))
    want = torch.zeros(V, d, device="cuda").index_add_(0, ids[[0, 1, 3]], g[[0, 1, 3]].float())
    assert torch.equal(inner.float(), want)  # whole numbers up to 183
    edge = base.clone()
    edge[off:off + V * ld].view(V, ld)[:, :d] = 7.0
    assert (edge == 7.0).all()


def test_a_gradient_of_few_tokens_is_not_slower_than_a_fill():
    """fp32, an odd vocabulary of odd width, where no row ends on a 16-byte boundary: a fill and an index_add_ take 261
    us, value-wise zeros made it 339, now 231."""
    from octopus_amd.embed_op import embed_bwd

    V, d, n = 151935, 2559, 8
    ids, g = torch.arange(n, device="cuda") * 1001, torch.randn(n, d, device="cuda")
    plain = _fastest(lambda: torch.zeros(V, d, device="cuda").index_add_(0, ids, g))
    assert _fastest(lambda: embed_bwd(g, ids, V)) <= 1.15 * plain
    assert torch.equal(embed_bwd(g, ids, V), torch.zeros(V, d, device="cuda").index_add_(0, ids, g))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_odd_widths_cost_about_what_even_ones_do(dtype):
    """The gradient of 1,501 tokens over [31,999, 1023] beside [32,000, 1024]: 95 and 26 us with loads that waited for
    each other, now 30 and 26; values that are no numbers stay in their columns, at the last one too."""
    from octopus_amd.embed_op import embed_bwd

    def one(V, d):
        ids, g = torch.arange(1501, device="cuda") * 17 % V, torch.ones(1501, d, dtype=dtype, device="cuda")
        return _fastest(lambda: embed_bwd(g, ids, V))

    assert one(31999, 1023) <= 2 * one(32000, 1024)
    ids, g = torch.tensor([1, 0, 1, 2], device="cuda"), torch.ones(4, 65, dtype=dtype, device="cuda")
    g[1, 64], g[3, 0], g[2, 63] = float("nan"), float("inf"), float("-inf")
    got = embed_bwd(g, ids, 3)
    want = torch.zeros(3, 65, device="cuda").index_add_(0, ids, g.float())
    assert torch.equal(got.float().nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [700, 5000, 100003])
@pytest.mark.parametrize("k", [1, 30, 65, 200])
def test_lists_of_few_values_above_a_run_of_equal_ones(dtype, V, k):
    """Allow-lists: fewer than k values above a mask of any value, none, one more than k; values and equal ones behind
    each other's columns; zeros of both signs; the oracle's lists, whole or in slices."""
    from octopus_amd.distill_op import head_topk

    g = torch.Generator().manual_seed(V + k)
    rows = []
    for mask in (-torch.inf, torch.finfo(dtype).min, -1e4, -0.3, 0.0, -0.0, 2.0):
        for kept in (0, 1, k - 1, k + 1):
            x = torch.full((V,), mask)
            at = torch.randperm(V, generator=g)[:min(kept, V - 1)]
            x[at] = 3.0 + torch.rand(len(at), generator=g)
            rows.append(x)
            below = x.clone()  # and below it, all over the row
            low = torch.randperm(V, generator=g)[:V // 2]
            below[low[x[low] < 2.5]] = -torch.inf
            rows.append(below)
    z = torch.stack(rows).to(dtype)
    want_ids, want = odist.topk(z, 1.0, k)
    for part in (slice(None), slice(0, 3)):  # three rows of 100,003: in slices where the type makes them long enough
        ids, logp = head_topk(z[part].cuda(), 1.0, k)
        assert torch.equal(ids.cpu(), want_ids[part])
        got, fin = logp.cpu().double(), want[part].isfinite()
        assert torch.equal(got == -torch.inf, want[part] == -torch.inf)
        # as tests/test_gpu_topk.py derives it
        assert ((got - want[part]).abs()[fin] <= 2e-5 + 2 ** -22 * want[part].abs()[fin]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [-torch.inf, -1e30])
def test_masked_rows_cost_a_second_sweep(dtype, mask):
    """512 rows of 151,936 with 10 unmasked logits each, k 64: below 6 times the time of unmasked rows (34 times as a
    radix select over one bin)."""
    from octopus_amd.distill_op import head_topk

    z = torch.randn(512, 151936, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    plain = _fastest(lambda: head_topk(z, 1.0, 64), calls=3)
    z[:, torch.arange(151936, device="cuda") % 15000 != 7] = mask
    assert _fastest(lambda: head_topk(z, 1.0, 64), calls=3) <= 6 * plain


@pytest.mark.parametrize("grad", [False, True])
def test_more_hidden_rows_than_a_launch_has_threads_for(grad):
    """2^24 rows and more, each a workgroup of 256 threads: the last rows' divergences and gradients are a small
    call's."""
    from octopus_amd.distill_op import fused_distill_head

    n, d, V, K, few = (1 << 24) + 5, 8, 9, 25, 70
    g = torch.Generator(device="cuda").manual_seed(8)
    h = torch.randn(n, d, generator=g, device="cuda").bfloat16().requires_grad_(grad)
    w = torch.randn(V, d, generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t = torch.randn(n, K, generator=g, device="cuda")
    loss, kl = fused_distill_head(h, w, ids, t, 1.0)
    last = h.detach()[-few:].clone().requires_grad_(True)
    few_loss, few_kl = fused_distill_head(last, w, ids[-few:], t[-few:], 1.0)
    assert torch.equal(kl[-few:], few_kl)
    assert abs(loss.item() - kl.double().sum().item()) <= 2.0 ** -23 * loss.item()
    if grad:
        (a,), (b,) = torch.autograd.grad(loss, h), torch.autograd.grad(few_loss, last)
        assert (a[-few:] - b).norm() <= 2 ** -7 * b.norm()  # stored exponentials and results of 16 bits, on both sides
        assert (a.float().norm(dim=1) > 0).all()


def test_a_confident_student_beside_its_list(monkeypatch):
    """bf16, one listed token of probability near 0 and a student that puts more than half of its mass on another: 0.3
    of dz's square are dense entries. Every entry that weighs takes one rounding and the gradient's own is the second,
    so its error is sqrt(2) times that of the exact gradient rounded, below sqrt(2.2). Dense entries rounded twice:
    sqrt(2.3)."""
    from octopus_amd import distill_op, head_op

    n, d, V = 400, 256, 16384
    g = torch.Generator().manual_seed(31)
    h = torch.randn(n, d, generator=g).to(torch.bfloat16)
    w = (torch.randn(V, d, generator=g) * 0.45).to(torch.bfloat16)
    ids, t = torch.randint(0, V, (n, 1), generator=g), torch.zeros(n, 1)
    rw = torch.rand(n, generator=g) + 0.5
    monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 1 << 62)
    monkeypatch.setattr(head_op, "_LATER_WORK", 1 << 62)
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    distill_op.fused_distill_head(hd, wd, ids.cuda(), t.cuda(), 1.0, rw.cuda())[0].backward()
    dz = odist.divergence(h.double() @ w.double().T, ids, t)[1] * rw.double()[:, None]
    assert dz.gather(1, ids).pow(2).sum() <= 0.7 * dz.pow(2).sum()
    for got, want in [(wd.grad, dz.T @ h.double()), (hd.grad, dz @ w.double())]:
        once = (want.to(torch.bfloat16).double() - want).norm()
        assert (got.cpu().double() - want).norm() <= 2.2 ** 0.5 * once


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_some_rows_of_more_than_2_gib(dtype):
    """Rows that take part, gathered from a hidden matrix past the 32-bit offsets of a mapped operand: the call of those
    rows by themselves, with and without gradients."""
    from octopus_amd.distill_op import fused_distill_head

    d, V, K = 2048, 1000, 6
    n = (1 << 31) // (d * dtype.itemsize) + 3000
    g = torch.Generator(device="cuda").manual_seed(9)
    h = torch.zeros(n, d, dtype=dtype, device="cuda")
    idx = torch.cat([torch.arange(0, n - 400, n // 100, device="cuda"), torch.arange(n - 300, n, device="cuda")])
    h[idx] = torch.randn(len(idx), d, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, d, generator=g, device="cuda") * 0.05).to(dtype)
    ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t, rw = torch.randn(n, K, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    count = torch.tensor([len(idx) - 5], dtype=torch.int32, device="cuda")
    part = idx[:-5]

    def run(h, idx, count, rows, grad):
        h, v = h.detach().requires_grad_(grad), w.detach().requires_grad_(grad)
        loss, kl = fused_distill_head(h, v, ids[rows], t[rows], 1.0, rw[rows], idx=idx, count=count)
        return loss.detach(), kl, *(torch.autograd.grad(loss, (h, v)) if grad else ())

    for grad in (False, True):
        got, want = run(h, idx, count, slice(None), grad), run(h[part], None, None, part, grad)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][part], want[1])
        rest = torch.ones(n, dtype=torch.bool, device="cuda").index_fill_(0, part, False)
        assert (got[1][rest] == 0).all()
        if grad:  # the same sums, over other tiles: a step of the type, or fp32's own
            step = torch.finfo(dtype).eps * (1 if dtype == torch.bfloat16 else 32)
            assert (got[2][part] - want[2]).norm() <= step * want[2].norm() and (got[2][rest] == 0).all()
            assert (got[3] - want[3]).norm() <= step * want[3].norm()


def test_a_later_weight_gradient_of_some_rows(monkeypatch):
    """The kept operands of rows that take part by idx and a count that changes after the call."""
    from octopus_amd import distill_op, head_op
    from octopus_amd.head_op import compact_rows

    n, d, V, K = 200, 256, 3000, 12
    h, w, ids, t = _small(n, d, V, K, seed=10)
    rw = torch.rand(n, generator=torch.Generator().manual_seed(11)).cuda()
    idx, count = compact_rows(torch.rand(n, generator=torch.Generator().manual_seed(12)).cuda() < 0.4)
    monkeypatch.setattr(head_op, "_LATER_SHARE", 1 << 20)
    out = []
    for later in (True, False):
        monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 0 if later else 1 << 62)
        monkeypatch.setattr(head_op, "_LATER_WORK", 1 << 62)
        assert (distill_op._later_bytes(h, w, idx, True, True) > 0) == later
        c = count.clone()
        loss, kl = distill_op.fused_distill_head(h, w, ids, t, 1.0, rw, idx=idx, count=c)
        c.fill_(3)
        out.append((loss.detach(), kl, *torch.autograd.grad(loss, (h, w))))
    a, b = out
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in zip(a[2:], b[2:]):
        assert (x - y).norm() <= 2 ** -8 * y.norm()  # the same products, split differently, and the result's rounding
