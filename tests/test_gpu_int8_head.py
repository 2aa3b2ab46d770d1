"""The head's logits from 8-bit integers (octopus_amd.int8_op.int8_head) and their gradients against 64 bits."""

import pytest
import torch

from octopus_amd import int8_op
from oracle import rows8 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(n, d, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(V, d, generator=g) * (2.5 / d ** 0.5)).to(dtype)
    return x, w


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _least(dtype):  # half a step below the normal numbers
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _check_logits(z, x, wq, ws, out):
    """The sum is exact; then its conversion and two products in fp32 (2^-24 each, to first order) and the rounding."""
    want = oracle.logits(x, wq.cpu(), ws.cpu())
    bound = (_half(out) + 4 * 2.0 ** -24) * want.abs() + _least(out)
    assert z.dtype == out and ((z.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,V", [(1, 64, 1000), (1, 2560, 515), (2, 16, 1), (3, 27, 5), (16, 1027, 300), (16, 4200, 100), (9, 4032, 700), (17, 128, 257),
                                   (33, 200, 255), (48, 4100, 131), (64, 1024, 512), (65, 130, 256), (130, 96, 1023), (256, 144, 300),
                                   (257, 1, 513), (300, 4097, 264), (129, 300, 515), (192, 65, 256), (193, 512, 511), (384, 97, 300), (400, 96, 513),
                                   (449, 2048, 260), (513, 200, 300), (600, 1100, 515), (1025, 64, 256),
                                   (800, 2048, 100)])
def test_logits(n, d, V, dtype):
    x, w = _inputs(n, d, V, dtype, n + d)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    _check_logits(int8_op.int8_head(x.to(DEV), wq, ws), x, wq, ws, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,V", [(129, 70, 33001), (192, 144, 33000), (193, 65, 33024), (256, 16, 32897), (257, 130, 22016),
                                   (300, 97, 22017), (385, 64, 17153), (449, 200, 17000), (600, 100, 14001),
                                   (1025, 48, 8000)])
def test_logits_of_wide_tiles(n, d, V, dtype):
    """More rows than 128 and more tiles of 128 x 128 than the card holds: tiles of 256 x 256 and narrower last ones."""
    x, w = _inputs(n, d, V, dtype, n + d)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    _check_logits(int8_op.int8_head(x.to(DEV), wq, ws), x, wq, ws, dtype)


@pytest.mark.parametrize("out", TYPES)
def test_other_types_and_shapes(out):
    x, w = _inputs(60, 72, 400, torch.bfloat16)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    z = int8_op.int8_head(x.to(DEV).view(3, 20, 72), wq, ws, out_dtype=out)
    assert z.shape == (3, 20, 400)
    _check_logits(z.view(60, 400), x, wq, ws, out)
    wide = torch.randn(60, 200).to(torch.bfloat16)
    for y in (wide[:, 3:75], wide[::3, :72], wide[:1, :72].expand(5, 72), wide[:72].t()[:60]):
        y = y[:, :72] if y.shape[1] >= 72 else torch.cat([y, y], 1)[:, :72]
        _check_logits(int8_op.int8_head(y.to(DEV), wq, ws, out_dtype=out), y, wq, ws, out)
    assert int8_op.int8_head(x.to(DEV)[:0], wq, ws).shape == (0, 400)


def test_largest_sums():
    """Rows and weights of nothing but the largest quotient: the sums reach 127^2 d."""
    d = 131072
    x = torch.ones(3, d)
    x[1] = -1
    wq = torch.full((300, d), 127, dtype=torch.int8, device=DEV)
    ws = torch.ones(300, device=DEV)
    z = int8_op.int8_head(x.to(DEV), wq, ws)
    _check_logits(z, x, wq, ws, torch.float32)
    with pytest.raises(ValueError):
        int8_op.int8_head(torch.ones(1, d + 16, device=DEV), torch.zeros(2, d + 16, dtype=torch.int8, device=DEV), ws[:2])


def test_rows_without_a_scale_and_odd_layouts():
    x, w = _inputs(20, 45, 70, torch.float32)
    x[3] = 0
    x[5, 7] = float("nan")
    x[6, 1] = float("inf")
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    z = int8_op.int8_head(x.to(DEV), wq, ws).cpu()
    assert (z[3] == 0).all() and torch.isnan(z[5]).all() and torch.isnan(z[6]).all()
    assert torch.isfinite(z[[0, 1, 2, 4, 7, 19]]).all()
    # weights whose rows are not padded, and padded with something else than zeros
    loose = wq.cpu().contiguous().to(DEV)
    full = torch.randint(-128, 127, (70, 64), dtype=torch.int8, device=DEV)
    full[:, :45] = wq
    for other in (loose, full[:, :45], wq.t().contiguous().t()):
        assert torch.equal(int8_op.int8_head(x.to(DEV), other, ws).cpu().nan_to_num(), z.nan_to_num())


def _bound_grads(g, x, wq, ws, dtype, out):
    gr, gw, mag_r, mag_w = oracle.grads(g, x, wq.cpu(), ws.cpu())
    n, V = g.shape
    def bound(res, mag, terms, other):
        # each 8-bit operand times its scale rounded once (fp32: three bf16 parts, 2^-22), the fp32 sum, the result
        per = max(_half(dtype), 2.0 ** -22) + (terms + 8) * 2.0 ** -24
        return mag * per + other * _least(dtype) + _half(out) * (res.abs() + mag * per) + _least(out)
    return gr, gw, bound(gr, mag_r, V, g.double().abs().sum(1, keepdim=True)), \
        bound(gw, mag_w, n, g.double().abs().sum(0)[:, None])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,V", [(1, 64, 100), (3, 27, 5), (17, 130, 257), (64, 256, 512), (70, 300, 1000), (257, 96, 515),
                                   (40, 512, 20000)])
def test_gradients(n, d, V, dtype):
    x, w = _inputs(n, d, V, dtype, n)
    g = (torch.randn(n, V, generator=torch.Generator().manual_seed(7)) / 8).to(dtype)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    gr, gw, bound_r, bound_w = _bound_grads(g, x, wq, ws, dtype, dtype)
    xd, wd, gd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True), g.to(DEV)
    for rows, weight in ((True, True), (True, False), (False, True)):
        z = int8_op.int8_head(xd if rows else xd.detach(), wq, ws, weight=wd if weight else None)
        wrt = [t for t, on in ((xd, rows), (wd, weight)) if on]
        got = list(torch.autograd.grad(z, wrt, gd))
        if rows:
            r = got.pop(0)
            assert r.dtype == dtype and ((r.cpu().double() - gr).abs() <= bound_r).all()
        if weight:
            assert got[0].dtype == dtype and ((got[0].cpu().double() - gw).abs() <= bound_w).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,V", [(1, 1, 1), (1, 300, 31), (2, 17, 5000), (15, 513, 33), (16, 256, 256), (17, 255, 20011),
                                   (31, 1027, 515), (32, 2560, 3001), (33, 40, 700), (128, 72, 300), (129, 300, 1000),
                                   (150, 96, 4001)])
def test_gradients_of_few_rows(n, d, V, dtype):
    """g off every 16-byte boundary, with no numbers around its rows; weights whose padding is not zeros."""
    x, w = _inputs(n, d, V, dtype, n + V)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    full = torch.full((V, wq.stride(0) if V > 1 else -(-d // 16) * 16), 77, dtype=torch.int8, device=DEV)
    full[:, :d] = wq
    store = torch.full((n, V + 7), float("nan"), dtype=dtype, device=DEV)
    g = (torch.randn(n, V, generator=torch.Generator().manual_seed(7)) / 8).to(dtype)
    store[:, 3:V + 3] = g.to(DEV)
    gr, gw, bound_r, bound_w = _bound_grads(g, x, wq, ws, dtype, dtype)
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    alone, = torch.autograd.grad(int8_op.int8_head(xd, full[:, :d], ws), xd, store[:, 3:V + 3])
    rows, weight = torch.autograd.grad(int8_op.int8_head(xd, full[:, :d], ws, weight=wd), (xd, wd), store[:, 3:V + 3])
    assert torch.equal(alone, rows) and ((rows.cpu().double() - gr).abs() <= bound_r).all()
    assert ((weight.cpu().double() - gw).abs() <= bound_w).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_strided_and_broadcast_g(dtype):
    n, d, V = 37, 48, 130
    x, w = _inputs(n, d, V, dtype)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    base = (torch.randn(2 * n, V + 9, generator=torch.Generator().manual_seed(1)) / 8).to(dtype)
    base = base.to(DEV)
    for g in (base[::2, 5:V + 5], base[:1, :V].expand(n, V), base[0, :1].expand(n, V),
              base[n:, 9:].t().contiguous().t()):
        gr, gw, bound_r, bound_w = _bound_grads(g.cpu(), x, wq, ws, dtype, dtype)
        z = int8_op.int8_head(xd, wq, ws, weight=wd)
        a, b = torch.autograd.grad(z, (xd, wd), g)
        assert ((a.cpu().double() - gr).abs() <= bound_r).all() and ((b.cpu().double() - gw).abs() <= bound_w).all()


@pytest.mark.parametrize("n", [1, 63, 64, 65, 130])
def test_gradients_of_g_read_where_it_lies(n):
    """16-bit g in whole chunks, its last row the end of its memory; the columns between its rows are no numbers."""
    d, V = 80, 264
    x, w = _inputs(n, d, V, torch.bfloat16)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    g = (torch.randn(n, V, generator=torch.Generator().manual_seed(n)) / 8).to(torch.bfloat16)
    gr, gw, bound_r, bound_w = _bound_grads(g, x, wq, ws, torch.bfloat16, torch.bfloat16)
    for ld, off in ((V, 0), (V + 8, 0), (V + 40, 24)):
        store = torch.full(((n - 1) * ld + V + off,), float("nan"), dtype=torch.bfloat16, device=DEV)
        at = store[off:].as_strided((n, V), (ld, 1))
        at.copy_(g)
        for rows, weight in ((True, True), (False, True), (True, False)):
            z = int8_op.int8_head(xd if rows else xd.detach(), wq, ws, weight=wd if weight else None)
            got = list(torch.autograd.grad(z, [t for t, on in ((xd, rows), (wd, weight)) if on], at))
            if rows:
                assert ((got.pop(0).cpu().double() - gr).abs() <= bound_r).all()
            if weight:
                assert ((got[0].cpu().double() - gw).abs() <= bound_w).all()


def test_gradients_of_other_types():
    """fp32 logits of bf16 rows and weights: gradients in the rows' and the weight's type."""
    x, w = _inputs(50, 64, 200, torch.bfloat16)
    g = torch.randn(50, 200, generator=torch.Generator().manual_seed(2)) / 8
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    gr, gw, bound_r, bound_w = _bound_grads(g, x, wq, ws, torch.float32, torch.bfloat16)
    xd, wd = x.to(DEV).view(5, 10, 64).requires_grad_(True), w.to(DEV).requires_grad_(True)
    z = int8_op.int8_head(xd, wq, ws, weight=wd, out_dtype=torch.float32)
    a, b = torch.autograd.grad(z, (xd, wd), g.view(5, 10, 200).to(DEV))
    assert a.dtype == b.dtype == torch.bfloat16 and a.shape == (5, 10, 64)
    assert ((a.cpu().double().view(50, 64) - gr).abs() <= bound_r).all()
    assert ((b.cpu().double() - gw).abs() <= bound_w).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 300])
def test_gradients_that_are_not_finite_stay_in_their_row_and_column(n, dtype):
    """As the formula has them: row r of the rows' gradient and row v of the weight's."""
    x, w = _inputs(n, 72, 520, dtype)
    w[7] = 0
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    g = torch.randn(n, 520, generator=torch.Generator().manual_seed(2)).to(dtype)
    g[1, 7], g[2, 515] = torch.nan, torch.inf
    xd = x.to(DEV).requires_grad_(True)
    wd = w.to(DEV).requires_grad_(True)
    int8_op.int8_head(xd, wq, ws, weight=wd).backward(g.to(DEV))
    rows, weights = torch.ones(n, dtype=torch.bool), torch.ones(520, dtype=torch.bool)
    rows[1] = rows[2] = False
    weights[7] = weights[515] = False
    for grad, fine in ((xd.grad.cpu(), rows), (wd.grad.cpu(), weights)):
        assert grad[fine].isfinite().all() and not grad[~fine].isfinite().any()


def test_fp32_gradients_keep_24_bits():
    """Each value of g alone: one nonzero product to a sum, so the error is that of the parts (2^-24 of the value, and
    of g times the scale) and of the result's rounding; over the range that three parts of normal numbers hold."""
    n, d, V = 64, 48, 64
    x, w = _inputs(n, d, V, torch.float32)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    size = torch.logspace(-28, 28, n, dtype=torch.float64)
    g = torch.diag((torch.rand(n, generator=torch.Generator().manual_seed(3), dtype=torch.float64) + 1) * size).float()
    xd = x.to(DEV).requires_grad_(True)
    wd = w.to(DEV).requires_grad_(True)
    int8_op.int8_head(xd, wq, ws, weight=wd).backward(g.to(DEV))
    rows, weights, *_ = oracle.grads(g, x, wq.cpu(), ws.cpu())
    for grad, want in ((xd.grad, rows), (wd.grad, weights)):
        assert ((grad.cpu().double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


def test_gradients_against_differences():
    """The rows' gradient against differences of the logits of the same 8-bit weights at rows that are not rounded."""
    x, w = _inputs(4, 32, 50, torch.float32)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    g = torch.randn(4, 50, generator=torch.Generator().manual_seed(4))
    xd = x.to(DEV).requires_grad_(True)
    (got,) = torch.autograd.grad(int8_op.int8_head(xd, wq, ws), xd, g.to(DEV))
    wide = oracle.widen(wq.cpu().long(), ws.cpu()[:, None])
    f = lambda t: (g.double() * (t @ wide.T)).sum().item()  # noqa: E731
    for r, k in [(0, 0), (1, 13), (3, 31)]:
        up, down = x.double().clone(), x.double().clone()
        up[r, k] += 1e-3
        down[r, k] -= 1e-3
        diff = (f(up) - f(down)) / 2e-3  # linear: off by fp64's rounding of f, 1e-16 x 100 / 1e-3
        assert abs(diff - got[r, k].item()) <= 1e-9 + 60 * 2.0 ** -22 * g[r].abs().sum().item() * wide.abs().max().item()


def test_changed_weights_and_second_derivatives_raise():
    x, w = _inputs(8, 32, 40, torch.bfloat16)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xd = x.to(DEV).requires_grad_(True)
    z = int8_op.int8_head(xd, wq, ws)
    wq.add_(0)
    with pytest.raises(RuntimeError, match="changed in place"):
        z.sum().backward()
    z = int8_op.int8_head(xd, wq, ws)
    c = torch.ones_like(z).requires_grad_(True)
    (gr,) = torch.autograd.grad(z, xd, c, create_graph=True)
    with pytest.raises(RuntimeError):
        gr.sum().backward()


def test_refusals():
    x, w = _inputs(4, 32, 40, torch.bfloat16)
    x, w = x.to(DEV), w.to(DEV)
    wq, ws = int8_op.quantise_rows(w)
    for args, kw in [((x[:, :31], wq, ws), {}), ((x, wq[0], ws), {}), ((x, wq.short(), ws), {}), ((x, wq, ws[:39]), {}),
                     ((x, wq, ws.half()), {}), ((x, wq, ws), {"weight": w[:39]}), ((x.cpu(), wq, ws), {}),
                     ((x, wq.cpu(), ws), {})]:
        with pytest.raises(ValueError):
            int8_op.int8_head(*args, **kw)
    for args, kw in [((x.double(), wq, ws), {}), ((x, wq, ws), {"out_dtype": torch.float64})]:
        with pytest.raises(NotImplementedError):
            int8_op.int8_head(*args, **kw)
