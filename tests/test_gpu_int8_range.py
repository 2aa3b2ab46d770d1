"""int8_head and its gradients where the first tests did not go: f16 logits of operands outside f16's range, dense
shares of many blocks of weight rows, saved rows that a hook gives back in another layout, tangents of forward mode,
many rows."""

import pytest
import torch

from octopus_amd import int8_op
from oracle import rows8 as oracle
from tests.test_gpu_int8_head import TYPES, _bound_grads, _check_logits, _half, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _f16_bound(ref, mag, terms, out, g_sums, scales):
    """The widened operand to f16's 11 bits, the fp32 sum, the result. The operand is widened times a power of two 2^k
    that brings the largest scale to 2^7 or more (2^-k <= 2^-7 of that scale); below 2^-14 its step is 2^-24, half of
    which is off by at most 2^-25 2^-k <= 2^-32 of the largest scale for each of g's values."""
    off = mag * (2.0 ** -11 + (terms + 8) * 2.0 ** -24) + g_sums * scales.max() * 2.0 ** -32
    return off + _half(out) * (ref.abs() + off) + torch.finfo(out).smallest_normal * torch.finfo(out).eps


def _check_f16(gr, gw, up, x, wq, ws, xs):
    """Each of gr, gw that is not None."""
    up, ws, xs = up.cpu(), ws.cpu().double(), xs.cpu().double()
    ref_r, ref_w, mag_r, mag_w = oracle.grads(up, x, wq.cpu(), ws)
    sums = up.double().abs()
    for got, ref, bound in ((gr, ref_r, lambda t: _f16_bound(ref_r, mag_r, sums.shape[1], t, sums.sum(1)[:, None],
                                                             ws[ws.isfinite()])),
                            (gw, ref_w, lambda t: _f16_bound(ref_w, mag_w, sums.shape[0], t, sums.sum(0)[:, None],
                                                             xs[xs.isfinite()]))):
        if got is not None:
            assert bool(((got.cpu().double() - ref).abs() <= bound(got.dtype)).all())


@pytest.mark.parametrize("n,d,V", [(9, 70, 600), (40, 96, 515), (200, 144, 640), (257, 65, 1027)])
@pytest.mark.parametrize("size", [1e5, 1e-7, 1e-30, 1e30])
@pytest.mark.parametrize("rows_dtype", [torch.bfloat16, torch.float32])
def test_f16_gradients_of_operands_outside_f16(rows_dtype, size, n, d, V):
    """f16 logits are finite where the rows' size and the weights' cancel; so are their gradients."""
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(n, d, generator=g) * size).to(rows_dtype)
    w = (torch.randn(V, d, generator=g) / size).to(rows_dtype)
    up = (torch.randn(n, V, generator=g) / 8).half()
    up[:, 1::7] = 0
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xd, wd = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    z = int8_op.int8_head(xd, wq, ws, weight=wd, out_dtype=torch.float16)
    _check_logits(z.detach(), x, wq, ws, torch.float16)
    gr, gw = torch.autograd.grad(z, (xd, wd), up.to(DEV))
    _check_f16(gr, gw, up, x, wq, ws, int8_op.quantise_rows(x.to(DEV))[1])


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("n,V", [(9, 700), (200, 700), (200, 16700), (20, 16700)])
def test_f16_gradients_of_rows_of_many_sizes(n, V, far):
    """Rows and weight rows between 2^-20 and 2^10, some of zeros: what is small beside the largest is off by a step
    that is small beside it. far: one row alone lies outside f16's numbers."""
    d = 80
    g = torch.Generator().manual_seed(3)
    x = torch.randn(n, d, generator=g) * torch.exp2(torch.randint(-20, 10, (n, 1), generator=g).float())
    w = torch.randn(V, d, generator=g) * torch.exp2(torch.randint(-20, 10, (V, 1), generator=g).float())
    x[1], w[2] = 0, 0
    if far:
        x[n // 2] *= 2.0 ** 24
        w[V * 9 // 16] *= 2.0 ** 24
    up = (torch.randn(n, V, generator=g) / 1024).half()
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xq, xs = int8_op.quantise_rows(x.to(DEV))
    gr, gw = int8_op.head_grads_i8(up.to(DEV), xq, xs, wq, ws, torch.float32, torch.float32, True, True)
    _check_f16(gr, gw, up, x, wq, ws, xs)


def test_f16_gradients_with_a_row_without_scale():
    """A row with a NaN is NaN in every weight's gradient (its values stand in every sum) and takes no other row's
    bits."""
    n, d, V = 200, 64, 520
    x, w = _inputs(n, d, V, torch.bfloat16)
    x[3, 5] = float("nan")
    up = (torch.randn(n, V, generator=torch.Generator().manual_seed(0)) / 8).half()
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xq, xs = int8_op.quantise_rows(x.to(DEV))
    gr, gw = int8_op.head_grads_i8(up.to(DEV), xq, xs, wq, ws, torch.float32, torch.float32, True, True)
    assert torch.isnan(gw).all()
    _check_f16(gr, None, up, x, wq, ws, xs)


# ---- dense shares of many blocks: a wave's later weight rows, the prefetch into them, the cut-off last block ---------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,V", [(1, 256, 151936), (17, 64, 70001), (32, 2560, 3001), (20, 4096, 70001),
                                   (32, 4800, 515)])
def test_few_rows_many_blocks(n, d, V, dtype):
    x, w = _inputs(n, d, V, dtype, n + d)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    _check_logits(int8_op.int8_head(x.to(DEV), wq, ws), x, wq, ws, dtype)


@pytest.mark.parametrize("n,d,V,dtype", [(8, 2560, 40003, torch.bfloat16), (8, 2560, 40003, torch.float16),
                                         (33, 1027, 60001, torch.bfloat16), (33, 1027, 60001, torch.float16),
                                         (16, 2304, 40003, torch.float32), (33, 1027, 60001, torch.float32)])
def test_few_rows_gradient_many_steps(n, d, V, dtype):
    x, w = _inputs(n, d, V, dtype, n)
    g = (torch.randn(n, V, generator=torch.Generator().manual_seed(7)) / 8).to(dtype)
    wq, ws = int8_op.quantise_rows(w.to(DEV))
    xq, xs = int8_op.quantise_rows(x.to(DEV))
    gr, _ = int8_op.head_grads_i8(g.to(DEV), xq, xs, wq, ws, dtype, dtype, True, False)
    want, _, bound, _ = _bound_grads(g, x, wq, ws, dtype, dtype)
    assert ((gr.cpu().double() - want).abs() <= bound).all()


# ---- what is saved, and what is not differentiated -------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 70, 200])
def test_saved_rows_in_another_layout(n):
    """A hook that gives the 8-bit rows back without the bytes between them: the same gradients."""
    x, w = _inputs(n, 45, 300, torch.bfloat16)
    up = (torch.randn(n, 300, generator=torch.Generator().manual_seed(1)) / 8).bfloat16().to(DEV)
    h, p = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    wq, ws = int8_op.quantise_rows(p)
    want = torch.autograd.grad(int8_op.int8_head(h, wq, ws, weight=p), (h, p), up)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        z = int8_op.int8_head(h, wq, ws, weight=p)
    got = torch.autograd.grad(z, (h, p), up)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_tangents_are_refused():
    """Forward mode has no derivative here: an error, not logits without their tangent."""
    import torch.autograd.forward_ad as fwad

    x, w = _inputs(6, 32, 50, torch.float32)
    x, w = x.to(DEV), w.to(DEV)
    wq, ws = int8_op.quantise_rows(w)
    for grad in (False, True):
        with fwad.dual_level():
            dual = fwad.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
            with pytest.raises((RuntimeError, NotImplementedError)):
                int8_op.int8_head(dual, wq, ws)
            with pytest.raises((RuntimeError, NotImplementedError)):
                int8_op.int8_head(x, wq, ws, weight=fwad.make_dual(w.clone(), torch.ones_like(w)))
    with fwad.dual_level():
        plain = int8_op.int8_head(x, wq, ws)  # no tangent: as ever
    assert torch.equal(plain, int8_op.int8_head(x, wq, ws))


# ---- many rows -------------------------------------------------------------------------------------------------------

def test_weight_gradient_of_two_million_rows():
    """A copy of g of 2^24 blocks and more, 121 GB beside g's 120: the first and the last rows alone."""
    n, d, V = 1 << 21, 16, 28673
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 250e9:
        pytest.skip("needs 250 GB of free memory")
    g = torch.zeros(n, V, dtype=torch.bfloat16, device=DEV)
    g[0, 0], g[-1, 0], g[-1, -1], g[n // 2, 7] = 2, 4, 8, 16
    xq = torch.ones(n, d, dtype=torch.int8, device=DEV)
    xq[-1], xq[n // 2, 3] = 5, 100
    xs = torch.full((n,), 0.5, device=DEV)
    wq, ws = torch.ones(V, d, dtype=torch.int8, device=DEV), torch.ones(V, device=DEV)
    try:
        _, gw = int8_op._grads(g, xq, xs, wq, ws, torch.bfloat16, torch.bfloat16, False, True)
        want = torch.zeros(V, d, device=DEV)
        want[0], want[-1], want[7] = 2 * 0.5 + 4 * 2.5, 8 * 2.5, 16 * 0.5
        want[7, 3] = 16 * 50
        assert torch.equal(gw.float(), want)
    finally:
        del g
        torch.cuda.empty_cache()
