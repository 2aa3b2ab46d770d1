"""head_topk against the 64-bit oracle: columns exactly, log-probabilities to fp32.

Tolerance of logp = (z - max) / T - ln S, per part: the product rounds by 2^-24 of itself; S is a sum of exponentials
whose arguments round by 2^-24 |t| (weighted by the exponential, below 2^-23 in all) and of up to 2^18 terms over 1,024
threads and a tree (about 200 roundings of 2^-24 at the worst, 1.2e-5); log2 adds 2^-23 |log2 S|."""

import math

import pytest
import torch

from oracle import distill as odist

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(z, T, k, view=None):
    from octopus_amd.distill_op import head_topk

    dev = z.cuda() if view is None else view(z)
    ids, logp = head_topk(dev, T, k)
    want_ids, want = odist.topk(z, T, k)
    assert ids.dtype == torch.int64 and logp.dtype == torch.float32
    assert torch.equal(ids.cpu(), want_ids)
    got = logp.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == -math.inf, want == -math.inf)
    fin = want.isfinite()
    err = (got - want).abs()[fin]
    assert (err <= 2e-5 + 2 ** -22 * want.abs()[fin]).all(), err.max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (3, 7, 7), (2, 64, 5), (5, 257, 256), (1, 1000, 64), (4, 4099, 20),
                                   (2, 32003, 128), (1, 151936, 64), (2, 151937, 256)])
def test_sizes(dtype, n, V, k):
    g = torch.Generator().manual_seed(n * V + k)
    _check((torch.randn(n, V, generator=g) * 3).to(dtype), 1.0 if V % 2 else 0.7, k)


@pytest.mark.parametrize("V", [20000, 100003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_orders(dtype, V):
    """Constant rows, few distinct values, ascending and descending rows, every large value in one thread's chunk, the
    same value at the list's end: rows that pass the candidates' room and rows that do not."""
    k = 64
    g = torch.Generator().manual_seed(3)
    rows = [torch.zeros(V), torch.full((V,), -2.5), torch.randint(0, 3, (V,), generator=g).float(),
            torch.linspace(-8, 8, V), torch.linspace(8, -8, V), torch.randn(V, generator=g)]
    rows[5][4096:4096 + 100] = torch.arange(100).float() + 10  # 100 neighbours above all others
    tied = torch.randn(V, generator=g).clamp(max=2.0)          # 450 values at the same maximum
    signed = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)  # zeros of both signs
    signed[7777] = 1.0
    few = torch.full((V,), -1.0)
    few[[19999, 3, 10000]] = torch.tensor([5.0, 5.0, 7.0])
    _check(torch.stack(rows + [tied, signed, few]).to(dtype), 1.0, k)


@pytest.mark.parametrize("V", [5000, 100003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_values(dtype, V):
    """Rows masked with -inf, with the type's lowest value, altogether so; NaN and +inf."""
    k = 30
    g = torch.Generator().manual_seed(4)
    z = torch.randn(9, V, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    z[0, 10:] = -math.inf          # 10 left
    z[1] = -math.inf
    z[2, 10:] = low
    z[3] = low
    z[4, ::2] = -math.inf
    z[5, 123] = math.nan
    z[6, [4, 4000]] = math.nan
    z[7, [9, 17]] = math.inf
    z[8, :4990] = low
    z[8, 4990:] = -math.inf
    _check(z, 1.0, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows(dtype):
    """Rows a step apart and off a 16-byte boundary; columns apart (copied)."""
    g = torch.Generator().manual_seed(5)
    z = (torch.randn(6, 3001, generator=g) * 2).to(dtype)

    def odd(x):
        base = torch.full((6, 3100), 99.0, dtype=dtype, device="cuda")
        base[:, 5:3006] = x.cuda()
        return base[:, 5:3006]

    _check(z, 1.0, 40, odd)
    _check(z, 1.0, 40, lambda x: x.T.contiguous().cuda().T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_and_many_rows(dtype):
    """Few rows are cut into slices, many are not: the same tokens, log-probabilities within twice the tolerance."""
    from octopus_amd.distill_op import head_topk

    z = (torch.randn(140, 100001, generator=torch.Generator().manual_seed(6)) * 2).to(dtype).cuda()
    z[5, 17:] = -math.inf
    z[6] = 0.25
    ids, logp = head_topk(z, 0.7, 100)
    for n in (1, 3, 40, 128):
        for r in (0, 5, 140 - n):
            few_ids, few = head_topk(z[r:r + n], 0.7, 100)
            assert torch.equal(few_ids, ids[r:r + n])
            fin = few.isfinite()
            assert torch.equal(fin, logp[r:r + n].isfinite())
            assert (few - logp[r:r + n])[fin].abs().max() <= 4e-5


def test_other_stream_and_graph():
    """On a side stream and replayed from a graph with other logits in place, each replay the eager call's bits."""
    from octopus_amd.distill_op import head_topk

    z = torch.randn(7, 32000, device="cuda").to(torch.bfloat16)
    want = head_topk(z, 1.0, 50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = head_topk(z, 1.0, 50)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = head_topk(z, 1.0, 50)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for s in range(3):
        z.copy_(torch.randn(7, 32000, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, head_topk(z, 1.0, 50)))


def test_refusals():
    from octopus_amd.distill_op import head_topk

    z = torch.randn(4, 100, device="cuda")
    for bad in [(z, 0.0, 5), (z, -1.0, 5), (z, 1.0, 0), (z, 1.0, 101), (z[0], 1.0, 5), (z.cpu(), 1.0, 5)]:
        with pytest.raises(ValueError):
            head_topk(*bad)
    with pytest.raises(ValueError):
        head_topk(torch.randn(2, 1000, device="cuda"), 1.0, 257)
    with pytest.raises(NotImplementedError):
        head_topk(z.double(), 1.0, 5)
    ids, logp = head_topk(z[:0], 1.0, 5)
    assert ids.shape == logp.shape == (0, 5)
