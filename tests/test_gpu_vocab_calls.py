"""Calls of the lists, the divergence and the embedding that their documentation allows beside the plain ones: rows of any
stride, second derivatives (refused), traces, another current stream, counts and scales of other types (refused)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_one_row_of_any_stride():
    """[V, 1] transposed: a row whose stride is 1."""
    from octopus_amd import distill_op, embed_op

    col = _r(700, 1)
    row = col.T
    assert row.stride(0) == 1
    a, b = distill_op.head_topk(row, 1.0, 9), distill_op.head_topk(row.clone(memory_format=torch.contiguous_format), 1.0, 9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ids, t = a
    z = row.detach().requires_grad_(True)
    kl = distill_op.distill_columns(z, 1.0, ids, t + 0.5)
    (grad,) = torch.autograd.grad(kl.sum(), z)
    assert grad.shape == (1, 700) and kl.isfinite().all()
    w = _r(16, 1, seed=1).T  # a vocabulary of one entry
    out = embed_op.embed_rows(w, torch.zeros(3, dtype=torch.int64, device="cuda"), 2.0)
    assert torch.equal(out, 2.0 * w.expand(3, 16))
    h = _r(64, 1, seed=2).to(torch.bfloat16).T
    weight = _r(300, 64, seed=3).to(torch.bfloat16)
    top = torch.arange(4, device="cuda")[None]
    a = distill_op.fused_distill_head(h, weight, top, torch.zeros(1, 4, device="cuda"), 1.0)
    b = distill_op.fused_distill_head(h.clone(memory_format=torch.contiguous_format), weight, top,
                                      torch.zeros(1, 4, device="cuda"), 1.0)
    assert torch.equal(a[0], b[0])


def test_second_derivatives_are_refused():
    """The backward passes are kernels without one of their own: asking for it raises, and is never a silent constant."""
    from octopus_amd import distill_op, embed_op

    z = _r(4, 200).requires_grad_(True)
    ids = torch.randint(0, 200, (4, 5), device="cuda")
    (g,) = torch.autograd.grad(distill_op.distill_columns(z, 1.0, ids, _r(4, 5)).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), z)
    w = _r(50, 16).requires_grad_(True)
    out = embed_op.embed_rows(w, ids)
    gout = _r(4, 5, 16, seed=4).requires_grad_(True)
    (g,) = torch.autograd.grad(out, w, gout, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), gout)
    h, weight = _r(4, 64).to(torch.bfloat16).requires_grad_(True), _r(200, 64).to(torch.bfloat16).requires_grad_(True)
    loss, _ = distill_op.fused_distill_head(h, weight, ids, _r(4, 5), 1.0)
    (g,) = torch.autograd.grad(loss, h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), h)


def test_backward_after_the_last_one_raises():
    from octopus_amd import distill_op

    h, weight = _r(4, 64).to(torch.bfloat16).requires_grad_(True), _r(200, 64).to(torch.bfloat16).requires_grad_(True)
    ids = torch.randint(0, 200, (4, 5), device="cuda")
    loss, _ = distill_op.fused_distill_head(h, weight, ids, _r(4, 5), 1.0)
    kept = torch.autograd.grad(loss, (h, weight), retain_graph=True)
    once = torch.autograd.grad(2 * loss, (h, weight))
    assert all(torch.equal(2 * a, b) for a, b in zip(kept, once))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (h, weight))


def test_without_gradients_the_forwards_workspace_is_enough():
    """The divergences alone, bit for bit those of the step, without the step's staging."""
    from octopus_amd import distill_op

    n, d, V = 600, 128, 40000
    h, weight = _r(n, d).to(torch.bfloat16), (_r(V, d, seed=1) * 0.2).to(torch.bfloat16)
    ids, t, rw = torch.randint(0, V, (n, 12), device="cuda"), _r(n, 12, seed=2), torch.rand(n, device="cuda")
    want = distill_op.fused_distill_head(h.clone().requires_grad_(True), weight, ids, t, 0.9, rw)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = distill_op.fused_distill_head(h, weight, ids, t, 0.9, rw)
    assert torch.cuda.max_memory_allocated() - before < n * V * 2  # no exponentials
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_traced_ops():
    """The registered ops: schemas, shapes under tracing and, where they have one, their gradients."""
    from octopus_amd import distill_op, embed_op

    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    z = _r(5, 300).requires_grad_(True)
    ids = torch.randint(0, 300, (5, 7), device="cuda")
    t = _r(5, 7, seed=5)
    torch.library.opcheck(distill_op.topk, (z.detach(), 1.0, 9), test_utils=tests)
    torch.library.opcheck(distill_op.distill_columns_fwd, (z, ids, t, 1.0, False), test_utils=tests)
    _, state, q = distill_op.distill_columns_fwd(z.detach(), ids, t, 1.0, False)
    torch.library.opcheck(distill_op.distill_columns_bwd, (z.detach(), ids, q, 1.0, state, t[:, 0]), test_utils=tests)
    w = _r(300, 64, seed=6).to(torch.bfloat16).requires_grad_(True)
    torch.library.opcheck(embed_op.embed_fwd, (w, ids, 2.0, -1), test_utils=tests)
    torch.library.opcheck(embed_op._embed_bwd, (_r(5, 7, 64), ids, 300, 2.0, -1, torch.float32), test_utils=tests)
    h = _r(5, 64, seed=7).to(torch.bfloat16).requires_grad_(True)
    torch.library.opcheck(distill_op.head_step_distill, (h, w, None, ids, t, None, None, None, 1.0, 1.0, 1.0, False, False,
                                                         True, True), test_utils=tests)
    loss, kl, gh, gw = distill_op.head_step_distill(h, w, None, ids, t, None, None, None, 1.0, 1.0, 1.0, False, False, True,
                                                    True)
    loss2, kl2 = distill_op.fused_distill_head(h, w, ids, t, 1.0)
    assert torch.equal(loss, loss2) and torch.equal(kl, kl2)
    for a, b in zip(torch.autograd.grad(3 * loss, (h, w), retain_graph=True), torch.autograd.grad(3 * loss2, (h, w))):
        assert torch.equal(a, b)
    assert torch.equal(gh, torch.autograd.grad(loss, h)[0])  # the op's own outputs stay as they were


def test_refused_companions():
    from octopus_amd import distill_op

    h, weight = _r(6, 64).to(torch.bfloat16), _r(200, 64).to(torch.bfloat16)
    ids, t = torch.randint(0, 200, (6, 5), device="cuda"), _r(6, 5)
    idx = torch.arange(6, device="cuda")
    count = torch.tensor([6], device="cuda")
    with pytest.raises(ValueError):
        distill_op.fused_distill_head(h, weight, ids, t, 1.0, idx=idx, count=count)
    q8 = weight.to(torch.float8_e4m3fn)
    for scale in (torch.ones(199, device="cuda"), torch.ones(200, dtype=torch.float64, device="cuda"), None):
        with pytest.raises(ValueError):
            distill_op.fused_distill_head(h, q8, ids, t, 1.0, w_scale=scale)
    for T in (float("nan"), float("inf"), 1e-39, 0.0):
        with pytest.raises(ValueError):
            distill_op.head_topk(h, T, 3)
    with pytest.raises(NotImplementedError):
        distill_op.fused_distill_head(h, q8.requires_grad_(True), ids, t, 1.0, w_scale=torch.ones(200, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_the_last_stay_as_they_were(dtype):
    """Outputs and in-place gradients lie inside larger buffers: nothing around them is written."""
    from octopus_amd import _lib
    from octopus_amd.embed_op import embed_grad_add_
    from octopus_amd.head_op import _DT, _p, _stream

    V, d, n = 37, 40, 90
    base = torch.full((V + 20, d + 24), 7.0, dtype=dtype, device="cuda")
    ids = torch.randint(0, V, (n,), device="cuda")
    embed_grad_add_(base[10:10 + V, 8:8 + d], _r(n, d).to(dtype), ids)
    edge = base.clone()
    edge[10:10 + V, 8:8 + d] = 7.0
    assert (edge == 7.0).all()
    # the dense gradient through the C ABI into rows a step apart: the gaps keep their values
    import ctypes

    out = torch.full((V + 2, d + 24), 7.0, dtype=dtype, device="cuda")
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_embed_bwd_workspace_bytes", n, V, d, ctypes.byref(nbytes))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device="cuda")
    g = _r(n, d, seed=1).to(dtype)
    inner = out[1:1 + V, 8:8 + d]
    _lib.call("octo_embed_bwd", _p(g), d, _DT[dtype], _p(ids), n, V, d, -1, 1.0, _p(inner), d + 24, _DT[dtype], 0, _p(ws),
              ws.numel(), _stream(g))
    edge = out.clone()
    edge[1:1 + V, 8:8 + d] = 7.0
    assert (edge == 7.0).all()
    want = torch.zeros(V, d, device="cuda").index_add_(0, ids, g.float())
    assert (inner.float() - want).abs().max() <= 2 ** -7 * want.abs().max()


def _head_inputs(seed, n=120, d=256, V=3003):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(n, d, generator=g, device="cuda").bfloat16().requires_grad_(True)
    w = (torch.randn(V, d, generator=g, device="cuda") * 0.1).bfloat16().requires_grad_(True)
    ids = torch.randint(0, V, (n, 20), generator=g, device="cuda")
    return h, w, ids, torch.randn(n, 20, generator=g, device="cuda"), torch.rand((), generator=g, device="cuda")


def _head_step(h, w, ids, t, c):
    from octopus_amd.distill_op import fused_distill_head

    loss, kl = fused_distill_head(h, w, ids, t, 0.9)
    return (kl, *torch.autograd.grad(loss, (h, w), c))


def _columns_step(h, w, ids, t, c):
    from octopus_amd.distill_op import distill_columns
    from octopus_amd.embed_op import embed_rows

    z = w.T[:100, :3001]  # any logits: 100 rows whose columns lie apart
    kl = distill_columns(z, 0.8, ids[:100], t[:100])
    out = embed_rows(w, ids, 2.0)
    return (kl.detach(), *torch.autograd.grad(kl, z, c.expand(100)), *torch.autograd.grad(out, w, torch.ones_like(out)))


@pytest.mark.parametrize("step", [_head_step, _columns_step])
@pytest.mark.parametrize("later", [False, True])
def test_captured_with_autograd(monkeypatch, step, later):
    """Forward and backward in one graph, replayed on new values between the program's own calls; later: the head's weight
    gradient made in the backward from kept operands."""
    from octopus_amd import head_op

    if later:
        monkeypatch.setattr(head_op, "_LATER_WEIGHTS", 0)
        monkeypatch.setattr(head_op, "_LATER_SHARE", 1 << 20)
    static = _head_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for seed in (1, 2, 3):
        new = _head_inputs(seed)
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(*new)))


def test_threads_with_streams_of_their_own():
    import threading

    inputs = [_head_inputs(k) for k in range(3)]
    want = [_head_step(*x) + _columns_step(*x) for x in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = _head_step(*inputs[k]) + _columns_step(*inputs[k])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_far_offsets():
    """A weight of more than 2^31 elements, logits of more than 2^32 bytes: the last rows."""
    from octopus_amd import distill_op, embed_op

    V, d = 1_100_000, 2048  # 2.25e9 elements
    w = torch.zeros(V, d, dtype=torch.bfloat16, device="cuda")
    w[-1] = 3.0
    w[-2] = torch.arange(d, device="cuda") % 128
    ids = torch.tensor([V - 1, V - 2, V, 0], device="cuda")
    got = embed_op.embed_rows(w, ids, 0.5)
    assert (got[0] == 1.5).all() and torch.equal(got[1], w[-2] * 0.5) and (got[2:] == 0).all()
    embed_op.embed_grad_add_(w, torch.ones(4, d, dtype=torch.bfloat16, device="cuda"), ids)
    assert (w[-1] == 4.0).all() and (w[0] == 1.0).all() and (w[1:-2].view(torch.int16) == 0).all()
    del w, got
    gw = embed_op.embed_bwd(torch.ones(4, d, dtype=torch.bfloat16, device="cuda"), ids, V)
    assert (gw[-2:] == 1).all() and (gw[0] == 1).all() and (gw[1:-2].view(torch.int16) == 0).all()
    del gw
    n, V = 18000, 128257  # 2.3e9 values of 16 bits
    z = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    z[-1, 5], z[-1, 128256], z[-2, 77] = 9.0, 9.0, 4.0
    top, logp = distill_op.head_topk(z, 1.0, 3)
    assert top[-1].tolist() == [5, 128256, 0] and top[-2].tolist() == [77, 0, 1]
    z.requires_grad_(True)
    kl = distill_op.distill_columns(z, 1.0, top, logp)
    (grad,) = torch.autograd.grad(kl.sum(), z)
    p = torch.softmax(z.detach()[-2:].double(), 1)
    q = torch.softmax(logp[-2:].double(), 1)
    want = p.scatter_add(1, top[-2:], -q)
    assert ((grad[-2:].double() - want).abs() <= 2 ** -8 * want.abs() + 1e-5 * (p + want.abs())).all()


def test_more_rows_than_a_launch_takes():
    """Rows past 2^21, tokens past 2^23: the last rows of the first launch, and the second's."""
    from octopus_amd import distill_op, embed_op

    n, V, K = (1 << 21) + 3, 8, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(n, V, generator=g, device="cuda").bfloat16()
    ids, logp = distill_op.head_topk(z, 1.0, K)
    kl = distill_op.distill_columns(z, 0.5, ids, logp)
    for part in (slice(0, 5), slice((1 << 21) - 4, None)):
        few, few_logp = distill_op.head_topk(z[part].clone(), 1.0, K)
        assert torch.equal(ids[part], few) and torch.equal(logp[part], few_logp)
        assert torch.equal(kl[part], distill_op.distill_columns(z[part].clone(), 0.5, few, few_logp))
    w = torch.randn(10, 8, generator=g, device="cuda").bfloat16()
    tokens = torch.randint(0, 10, ((1 << 23) + 5,), generator=g, device="cuda")
    assert torch.equal(embed_op.embed_rows(w, tokens), w[tokens])


def test_a_strided_weight_scale():
    """fp8 weights whose scales lie apart."""
    from octopus_amd import distill_op

    n, d, V, K = 5, 64, 200, 4
    g = torch.Generator(device="cuda").manual_seed(4)
    h = torch.randn(n, d, generator=g, device="cuda").bfloat16()
    W = torch.randn(V, d, generator=g, device="cuda").to(torch.float8_e4m3fn)
    scale = torch.rand(V, 2, generator=g, device="cuda")[:, 0]
    ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t = torch.randn(n, K, generator=g, device="cuda")
    got, want = (distill_op.fused_distill_head(h, W, ids, t, 1.0, w_scale=s)[1] for s in (scale, scale.contiguous()))
    assert torch.equal(got, want)


def test_broadcast_inputs():
    """One hidden row, one row of logits and one weight shared by all: the gradients add up over what shares them."""
    from octopus_amd import distill_op, embed_op

    n, d, V, K = 6, 64, 200, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t = torch.randn(n, K, generator=g, device="cuda")
    W = torch.randn(V, d, generator=g, device="cuda")
    h, z = torch.randn(1, d, generator=g, device="cuda"), torch.randn(1, V, generator=g, device="cuda")
    tokens, up = torch.randint(0, V, (9,), generator=g, device="cuda"), torch.randn(9, d, generator=g, device="cuda")

    def grad(x, f):
        x = x.clone().requires_grad_(True)
        f(x).backward()
        return x.grad

    for x, shape, f in [(h, (n, d), lambda a: distill_op.fused_distill_head(a, W, ids, t, 1.0)[0]),
                        (z, (n, V), lambda a: distill_op.distill_columns(a, 1.0, ids, t).sum()),
                        (W[:, :1], (V, d), lambda a: (embed_op.embed_rows(a, tokens) * up).sum())]:
        shared, each = grad(x, lambda a: f(a.expand(shape))), grad(x.expand(shape).contiguous(), f)
        each = each.double().sum_to_size(x.shape)
        # sums of at most 64 fp32 values: 63 roundings of what they add up to at most
        bound = 64 * 2.0 ** -24 * grad(x.expand(shape).contiguous(), f).abs().double().sum_to_size(x.shape)
        assert ((shared.double() - each).abs() <= bound).all()


def test_reads_only_what_it_wrote():
    """Workspaces and outputs full of NaN and -1 beforehand: lists in slices, the divergence, the embedding's sort with
    tokens left out."""
    from octopus_amd import distill_op, embed_op
    from tests.test_gpu_poisoned import poisoned

    z = _r(3, 60001, seed=1)
    ids = torch.randint(-40, 700, (1501,), generator=torch.Generator().manual_seed(2)).cuda()
    up = _r(1501, 72, seed=3).bfloat16()
    into = _r(700, 72, seed=4).bfloat16()

    def run():
        lists = distill_op.head_topk(z, 0.7, 20)
        s = z.clone().requires_grad_(True)
        kl = distill_op.distill_columns(s, 0.7, *lists)
        dz, = torch.autograd.grad(kl.sum(), s)
        return (*lists, kl.detach(), dz, embed_op.embed_rows(into, ids), embed_op.embed_bwd(up, ids, 700, 0.5),
                embed_op.embed_grad_add_(into.clone(), up, ids, padding_idx=7))

    want = run()
    with poisoned():
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_row_taken_twice(dtype):
    """idx may name a row again (a run, as row lists of a packed stream do): the row counts as often."""
    from octopus_amd import distill_op

    n, d, V, K = 9, 64, 300, 5
    h, W = _r(n, d, seed=1).to(dtype), (_r(V, d, seed=2) * 0.3).to(dtype)
    ids = torch.randint(0, V, (n, K), generator=torch.Generator().manual_seed(3)).cuda()
    t = _r(n, K, seed=4)
    idx = torch.tensor([0, 2, 2, 2, 5, 8, 8], device="cuda")
    times = torch.bincount(idx, minlength=n).float()

    def run(**kw):
        hd, Wd = h.clone().requires_grad_(True), W.clone().requires_grad_(True)
        loss, kl = distill_op.fused_distill_head(hd, Wd, ids, t, 1.0, **kw)
        loss.backward()
        return loss.detach(), kl, hd.grad, Wd.grad

    got, want = run(idx=idx), run(row_weight=times)
    assert abs(got[0] - want[0]) <= 2.0 ** -22 * want[0]  # fp32 of a sum in 64 bits of kl's own bits
    assert torch.equal(got[1], want[1] * (times > 0))
    # bf16 and f16: both sides round the stored exponential and the result, and h^T with a scale of their own: four
    # roundings of half a unit that are not shared; fp32: products of 300 and 9 terms in other orders
    half = 300 * 2.0 ** -24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for a, b in zip(got[2:], want[2:]):
        assert (a.double() - b.double()).norm() <= 4 * half * b.double().norm()
