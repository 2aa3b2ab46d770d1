"""The 8-bit head, the held rows and the verification as a program uses them: together, captured, from threads and
streams, traced, over poisoned memory, in inference mode, over far offsets."""

import threading

import pytest
import torch

from octopus_amd import int8_op, verify_op
from oracle import distill as odist
from oracle import grpo as ogrpo
from oracle import rows8 as orows
from oracle import verify as overify

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(seed, n=70, d=272, V=3008, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(n, d, generator=g, device=DEV).to(dtype).requires_grad_(True)
    w = (torch.randn(V, d, generator=g, device=DEV) * 0.15).to(dtype).requires_grad_(True)
    up = (torch.randn(n, V, generator=g, device=DEV) / n).to(dtype)
    drafts = torch.randint(0, V, (n // 5, 4), generator=g, device=DEV)
    return h, w, up, drafts, torch.rand(n // 5, 5, generator=g, device=DEV)


def _step(h, w, up, drafts, u):
    """Weights and rows to 8 bits, logits, gradients, drafts checked, rows held and read back."""
    wq, ws = int8_op.quantise_rows(w)
    z = int8_op.int8_head(h, wq, ws, weight=w)
    gh, gw = torch.autograd.grad(z, (h, w), up)
    S, K = drafts.shape
    target = z.detach()[:S * (K + 1)].view(S, K + 1, -1)
    said = verify_op.verify_drafts(target, drafts, u, 0.9, draft_logits=target[:, :K].flip(0))
    best = verify_op.verify_drafts(target, drafts, None, 0.9, greedy=True)
    q, s = int8_op.quantise_rows(h, 64)
    return (z.detach(), gh, gw, *said, *best, s, int8_op.widen_rows(q, s, h.dtype, 64))


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_rollout_and_update():
    """Logits of an 8-bit policy, drafts verified on them, their log-probabilities the behaviour logprobs of the GRPO step
    on the full-precision head; then the student's divergence from the 8-bit teacher's lists."""
    from octopus_amd.distill_op import distill_columns, head_topk
    from octopus_amd.head_op import fused_grpo_head

    S, K, d, V, T = 12, 3, 128, 1500, 0.8
    g = torch.Generator().manual_seed(11)
    h = torch.randn(S * (K + 1), d, generator=g).to(torch.bfloat16)
    w = (torch.randn(V, d, generator=g) * 0.2).to(torch.bfloat16)
    u = torch.rand(S, K + 1, generator=g)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    z = int8_op.int8_head(h.to(DEV), wq, ws, out_dtype=torch.float32).view(S, K + 1, V)
    draft = z[:, :K].bfloat16().float() + 0.5 * torch.randn(S, K, V, generator=g).to(DEV)
    x = torch.multinomial(torch.softmax(draft.cpu() / T, 2).view(S * K, V), 1, generator=g).view(S, K)
    tokens, accepted, logp = verify_op.verify_drafts(z, x.to(DEV), u.to(DEV), T, draft_logits=draft)
    want, count, lp = overify.verify_dense(z.cpu(), x, u, T, draft.cpu())
    assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), count)
    assert (accepted > 0).any() and (accepted < K).any()
    torch.testing.assert_close(logp.cpu().double(), lp, rtol=2.0 ** -24, atol=1e-12)

    mask = (tokens >= 0).float().view(-1)
    adv = torch.randn(S * (K + 1), generator=g).to(DEV)
    hd, wd = h.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    loss, cols = fused_grpo_head(hd, wd, tokens.view(-1).clamp(min=0), T, adv, mask, old=logp.view(-1))
    loss.backward()
    lo, _ = ogrpo.grpo(cols[:, 0].cpu().double().numpy(), adv.cpu().numpy(), mask.cpu().numpy(), prox=None,
                       old=logp.view(-1).cpu().double().numpy())
    assert abs(loss.item() - lo) <= 1e-5 * max(1.0, abs(lo)) and hd.grad.isfinite().all()
    # the 8-bit policy's logprobs lie near the full-precision head's: the rounding of 8 bits moves a logit by a few
    # hundredths of its spread of about 2.3 / 0.8
    assert ((cols[:, 0] - logp.view(-1)) * mask).abs().max() < 0.5

    ids, teacher = head_topk(z.view(-1, V), T, 16)
    hs, wm = h.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    sq, ss = int8_op.quantise_rows(wm)
    kl = distill_columns(int8_op.int8_head(hs, sq, ss, weight=wm, out_dtype=torch.float32), 1.0, ids, teacher)
    kl.mean().backward()
    zz = orows.logits(h, sq.cpu(), ss.cpu())
    want_kl, dz = odist.divergence(zz, ids.cpu(), teacher.cpu())
    assert (kl.detach().cpu().double() - want_kl).abs().max() <= 1e-4
    gr, gw, mag_r, mag_w = orows.grads(dz / dz.shape[0], h, sq.cpu(), ss.cpu())
    # fp32 logits and gradients of them (a few 2^-22 each), then one rounding to bf16
    for got, ref, mag in ((hs.grad, gr, mag_r), (wm.grad, gw, mag_w)):
        assert ((got.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5 * mag + 1e-30).all()


def test_captured_with_autograd():
    """Weights quantised, both passes and both verifications in one graph, replayed on new values between the program's
    own calls."""
    static = _inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(*static)
    for seed in (1, 2, 3):
        new = _inputs(seed)
        with torch.no_grad():
            for a, b in zip(static, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert _same(got, _step(*new))


def test_two_graphs_in_turn():
    """Graphs with workspaces of their own, replayed in turn and on two streams at once; the many-logits route too."""
    g = torch.Generator(device=DEV).manual_seed(4)
    made = []
    for k in range(2):
        z = torch.randn(300, 2, 30000, generator=g, device=DEV).bfloat16()
        x = torch.randint(0, 30000, (300, 1), generator=g, device=DEV)
        u = torch.rand(300, 2, generator=g, device=DEV)
        want = [t.clone() for t in verify_op.verify_drafts(z, x, u, 1.0)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = verify_op.verify_drafts(z, x, u, 1.0)
        # the inputs stay with the graph that reads them: the next capture gives freed memory back to the device
        made.append((graph, got, want, torch.cuda.Stream(), (z, x, u)))
    for _ in range(3):
        for _, got, *_ in made:
            for t in got:
                t.fill_(-7)
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(_same(got, want) for _, got, want, _, _ in made)


def test_threads_with_streams_of_their_own():
    inputs = [_inputs(k) for k in range(3)]
    want = [_step(*x) for x in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = _step(*inputs[k])
                torch.cuda.current_stream().synchronize()
                if not _same(got, want[k]):
                    wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("n", [5, 70, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_reads_only_what_it_wrote(n, dtype):
    from tests.test_gpu_poisoned import poisoned

    inputs = _inputs(n, n, 136, 2001, dtype)
    want = _step(*inputs)
    with poisoned():
        got = _step(*inputs)
    assert _same(got, want)


def test_many_logits_over_poisoned_memory():
    from tests.test_gpu_poisoned import poisoned

    g = torch.Generator(device=DEV).manual_seed(6)
    z = torch.randn(400, 3, 20000, generator=g, device=DEV).bfloat16()
    z[7] = float("nan")
    zd = (z[:, :2].float() + 0.3 * torch.randn(400, 2, 20000, generator=g, device=DEV)).bfloat16()
    x, u = zd.float().argmax(2), torch.rand(400, 3, generator=g, device=DEV)
    n = torch.randint(0, 3, (400,), generator=g, device=DEV)
    run = lambda: verify_op.verify_drafts(z, x, u, 1.1, draft_logits=zd, lengths=n)  # noqa: E731
    want = run()
    with poisoned():
        got = run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(got[2].nan_to_num(), want[2].nan_to_num())


def test_traced_ops():
    """The registered ops: schemas, shapes under tracing, gradients; and the public calls inside a trace."""
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    h, w, up, drafts, u = _inputs(1, 20, 40, 300)
    wq, ws = int8_op.quantise_rows(w)
    torch.library.opcheck(int8_op._quantise_op, (h.detach(), 0), test_utils=tests)
    torch.library.opcheck(int8_op._quantise_op, (h.detach().view(4, 5, 40), 32), test_utils=tests)
    torch.library.opcheck(int8_op._widen_op, (wq, ws, torch.bfloat16, 0), test_utils=tests)
    torch.library.opcheck(int8_op.head_logits_i8, (h, wq, ws, w, torch.float32), test_utils=tests)
    z, xq, xs = int8_op.head_logits_i8(h, wq, ws, w, torch.bfloat16)
    torch.library.opcheck(int8_op.head_grads_i8, (up, xq, xs, wq, ws, torch.bfloat16, torch.bfloat16, True, True),
                          test_utils=tests)
    target = z.detach().view(4, 5, 300)
    torch.library.opcheck(verify_op._verify_op, (target, drafts, u, target[:, :4], None, 1.0, False), test_utils=tests)
    plain = int8_op.int8_head(h, wq, ws, weight=w)
    assert torch.equal(z, plain)
    assert _same(torch.autograd.grad(z, (h, w), up, retain_graph=True), torch.autograd.grad(plain, (h, w), up))
    with pytest.raises(RuntimeError, match="only the logits"):
        torch.autograd.grad(xs.sum(), h)

    def run(h, w):
        q, s = int8_op.quantise_rows(w)
        z = int8_op.int8_head(h, q, s, weight=w)
        said = verify_op.verify_drafts(z.view(4, 5, 300), drafts, u, 1.0)
        return (z, *said, int8_op.widen_rows(q, s, torch.float32))

    got = torch.compile(run, backend="aot_eager", fullgraph=True)(h, w)
    want = run(h, w)
    assert _same(got, want)
    assert _same(torch.autograd.grad(got[0], (h, w), up), torch.autograd.grad(want[0], (h, w), up))


def test_inference_mode_and_saved_tensor_hooks():
    h, w, up, drafts, u = _inputs(2)
    with torch.inference_mode():
        wq, ws = int8_op.quantise_rows(w)
        z = int8_op.int8_head(h, wq, ws)
    z2 = int8_op.int8_head(h, wq, ws)  # weights made in inference mode, under autograd
    assert torch.equal(z, z2)
    (gh,) = torch.autograd.grad(z2, h, up)
    packed = []

    def pack(t):
        packed.append((t.dtype, t.numel()))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
        z3 = int8_op.int8_head(h, wq, ws, weight=w)
    again, _ = torch.autograd.grad(z3, (h, w), up)
    assert torch.equal(again, gh)
    assert packed == [(torch.int8, h.numel()), (torch.float32, h.shape[0])]  # 8 bits of the rows, no weight


def test_broadcast_rows_and_shared_weights():
    """One row for all, and a weight that two heads share: gradients add up over what shares them."""
    h, w, up, *_ = _inputs(3, 6, 64, 304, torch.float32)
    wq, ws = int8_op.quantise_rows(w)
    one = h.detach()[:1].clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(int8_op.int8_head(one.expand(6, 64), wq, ws), one, up)
    each = h.detach()[:1].expand(6, 64).contiguous().requires_grad_(True)
    (g6,) = torch.autograd.grad(int8_op.int8_head(each, wq, ws), each, up)
    assert ((g1 - g6.sum(0, keepdim=True)).abs() <= 6 * 2.0 ** -23 * g6.abs().sum(0)).all()
    two = int8_op.int8_head(h, wq, ws, weight=w).sum() + 2 * int8_op.int8_head(h, wq, ws, weight=w).sum()
    (gw,) = torch.autograd.grad(two, w)
    (ones,) = torch.autograd.grad(int8_op.int8_head(h, wq, ws, weight=w).sum(), w)
    assert torch.equal(gw, ones + 2 * ones)


def test_outputs_stay_inside():
    """The C calls write the rows and columns they are told to and nothing around them."""
    import ctypes

    from octopus_amd import _lib
    from octopus_amd.head_op import _p, _stream

    n, d, V = 40, 50, 301
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(n, d, generator=g, device=DEV).bfloat16()
    w = torch.randn(V, d, generator=g, device=DEV).bfloat16()
    wq, ws = int8_op.quantise_rows(w)
    for rows in (n, 7):
        z = torch.full((n + 2, V + 9), 7.0, dtype=torch.bfloat16, device=DEV)
        xq = torch.full((n + 1, 80), 77, dtype=torch.int8, device=DEV)
        xs = torch.full((n + 1,), 7.0, device=DEV)
        _lib.call("octo_head_logits_i8", _p(x), d, _lib.BF16, _p(wq), 64, _p(ws), rows, d, V, _p(xq), 80, _p(xs),
                  _p(z[1:, 3:]), V + 9, _lib.BF16, _stream(x))
        edge = z.clone()
        edge[1:1 + rows, 3:3 + V] = 7.0
        assert (edge == 7.0).all() and (xs[rows:] == 7.0).all() and (xq[rows:] == 77).all()
        assert (xq[:rows, 64:] == 77).all() and (xq[:rows, 50:64] == 0).all()
        assert torch.equal(z[1:1 + rows, 3:3 + V], int8_op.int8_head(x[:rows], wq, ws))
    up = torch.randn(n, V, generator=g, device=DEV).bfloat16()
    gr = torch.full((n + 2, d + 6), 7.0, dtype=torch.bfloat16, device=DEV)
    gw = torch.full((V + 2, d + 6), 7.0, device=DEV)
    xq, xs = int8_op.quantise_rows(x)
    size = ctypes.c_size_t(0)
    _lib.call("octo_head_grads_i8_workspace_bytes", _p(up), V, _lib.BF16, n, d, V, 1, 1, ctypes.byref(size))
    ws_ = torch.empty(size.value, dtype=torch.uint8, device=DEV)
    _lib.call("octo_head_grads_i8", _p(up), V, _lib.BF16, _p(xq), 64, _p(xs), _p(wq), 64, _p(ws), n, d, V,
              _p(gr[1:, 3:]), d + 6, _lib.BF16, _p(gw[1:, 3:]), d + 6, _lib.F32, _p(ws_), ws_.numel(), _stream(x))
    for t, inner in ((gr, (n, d)), (gw, (V, d))):
        edge = t.clone()
        assert not (edge[1:1 + inner[0], 3:3 + inner[1]] == 7.0).all()
        edge[1:1 + inner[0], 3:3 + inner[1]] = 7.0
        assert (edge == 7.0).all()


def test_far_offsets():
    """Weights of more than 2^31 bytes, logits of more than 2^31 values, held rows of more than 2^31."""
    V, d = (1 << 21) - 5, 1040
    wq = torch.zeros(V, d, dtype=torch.int8, device=DEV)
    wq[-1], wq[-2, 7], wq[0, 3] = 3, 100, -5
    ws = torch.full((V,), 0.5, device=DEV)
    for n in (3, 40, 150, 1100):
        x = torch.zeros(n, d, device=DEV)
        x[:, 7] = 127.0
        x[-1] = 127.0
        z = int8_op.int8_head(x.bfloat16(), wq, ws)
        assert z[-1, -1] == torch.tensor(127 * 3 * d * 0.5).bfloat16() and z[0, -1] == torch.tensor(127 * 3 * 0.5).bfloat16()
        assert (z[:, -2] == 127 * 100 * 0.5).all() and z[-1, 0] == torch.tensor(-5 * 127 * 0.5).bfloat16()
        assert z[:, 1:-2].abs().max() == 0
        del z
    del wq
    rows, d = 1_100_000, 2048
    x = torch.ones(rows, d, dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.arange(d, device=DEV) % 128
    q, s = int8_op.quantise_rows(x, 128)
    back = int8_op.widen_rows(q, s, torch.bfloat16, 128)
    assert (q[:-1] == 127).all() and torch.equal(back[-1], x[-1]) and torch.equal(back[-2], x[-2])


def test_gradients_over_far_offsets():
    """Weights of more than 2^31 bytes and gradients of more than 2^31 values: the first and the last rows alone."""
    V, d = (1 << 21) - 8, 1040
    wq = torch.zeros(V, d, dtype=torch.int8, device=DEV)
    wq[-1], wq[-2, 7], wq[0, 3] = 3, 100, -5
    ws = torch.full((V,), 0.5, device=DEV)
    for n in (3, 40, 1100):
        g = torch.zeros(n, V, dtype=torch.bfloat16, device=DEV)
        g[0, 0], g[-1, -1], g[-1, -2] = 2, 4, 8
        x = torch.ones(n, d, dtype=torch.bfloat16, device=DEV)
        xq, xs = int8_op.quantise_rows(x)
        rows, weight = int8_op._grads(g, xq, xs, wq, ws, torch.float32, torch.bfloat16, True, n == 40)
        want = torch.zeros(n, d, device=DEV)
        want[0, 3] = -5.0
        want[-1] = 6.0
        want[-1, 7] += 400.0
        assert torch.equal(rows, want)
        if weight is not None:
            assert (weight[0] == 2).all() and (weight[-1] == 4).all() and (weight[-2] == 8).all()
            assert not weight[1:-2].any()
        del g, weight


def test_verify_far_offsets():
    S, K, V = 700, 7, 400000  # 2.2e9 logits
    g = torch.Generator(device=DEV).manual_seed(2)
    z = torch.zeros(S, K + 1, V, dtype=torch.bfloat16, device=DEV)
    for r in range(0, S, 100):
        z[r:r + 100] = torch.randn(100, 1, V, generator=g, device=DEV).bfloat16()
    z[:, :, 17] = 25.0
    x = torch.full((S, K), 17, device=DEV)
    x[::3, 4] = 18
    u = torch.rand(S, K + 1, generator=g, device=DEV)
    tokens, accepted, logp = verify_op.verify_drafts(z, x, u, 1.0)
    for s in (0, 1, 350, 698, 699):
        want, count, lp = overify.verify_dense(z[s:s + 1].cpu(), x[s:s + 1].cpu(), u[s:s + 1].cpu(), 1.0)
        assert torch.equal(tokens[s:s + 1].cpu(), want) and torch.equal(accepted[s:s + 1].cpu(), count)
        torch.testing.assert_close(logp[s:s + 1].cpu().double(), lp, rtol=2.0 ** -24, atol=4e-6)
    small = verify_op.verify_drafts(z[695:].clone(), x[695:], u[695:], 1.0)
    assert torch.equal(small[0], tokens[695:]) and torch.equal(small[1], accepted[695:])


def test_more_sequences_than_a_launch_takes():
    """65,535 rows of a grid's second dimension: sequences in several launches."""
    S, K, V = 30000, 2, 40
    g = torch.Generator(device=DEV).manual_seed(3)
    z = torch.randn(S, K + 1, V, generator=g, device=DEV)
    zd = z[:, :K] + 0.5 * torch.randn(S, K, V, generator=g, device=DEV)
    x, u = torch.randint(0, V, (S, K), generator=g, device=DEV), torch.rand(S, K + 1, generator=g, device=DEV)
    n = torch.randint(0, K + 1, (S,), generator=g, device=DEV)
    got = verify_op.verify_drafts(z, x, u, 1.0, draft_logits=zd, lengths=n)
    for part in (slice(0, 50), slice(13090, 13130), slice(26200, 26230), slice(S - 20, S)):
        want = overify.verify_dense(z[part].cpu(), x[part].cpu(), u[part].cpu(), 1.0, zd[part].cpu(), n[part].cpu())
        assert torch.equal(got[0][part].cpu(), want[0]) and torch.equal(got[1][part].cpu(), want[1])
