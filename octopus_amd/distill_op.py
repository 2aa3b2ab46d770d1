"""Distillation from a teacher's top logits, over libocto_head.so.

    head_topk                          the teacher's list: the k largest logits of a row and their log-probabilities
    octohead::distill_columns_fwd/bwd  the student's divergence from the lists over materialised logits

A row's list is K slots (ids[r, k], teacher[r, k]): tokens, and the teacher's logits or log-probabilities of them, as
head_topk gives them. A slot whose id lies outside [0, V) or whose teacher value is -inf is empty (shorter lists), and the
same token may stand in several slots. With q the softmax of the teacher's values over a row's slots and p = softmax(z /
T) the student's distribution over the whole vocabulary,

    kl_r = sum_k q_k (log q_k - log p_ids[k])                             (a row without a slot: 0)
    dL/dz_v = g_r (Q p_v - sum of q_k over the slots of v) / T,  Q = sum q,  g_r = dL/dkl_r.

HIP tensors only; all work is queued on the current stream of the tensors' device, nothing synchronises with the host.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib
from .embed_op import _float_rows, _ids, _on_gpu
from .head_op import _DT, _p, _stream


def _lists(ids: Tensor, teacher: Tensor, rows: int) -> tuple[Tensor, Tensor]:
    if ids.dim() != 2 or ids.shape != teacher.shape or ids.shape[0] != rows:
        raise ValueError(f"octohead: lists [{rows}, K] expected, got ids {tuple(ids.shape)} and teacher "
                         f"{tuple(teacher.shape)}")
    if not 1 <= ids.shape[1] <= _lib.LIST_MAX:
        raise ValueError(f"octohead: lists of 1 to {_lib.LIST_MAX} slots, got {ids.shape[1]}")
    return _ids(ids), teacher.float().contiguous()


def _inv_T(temperature: float) -> float:
    if not temperature > 0:
        raise ValueError("temperature must be positive")
    return 1.0 / float(temperature)


# ---- the teacher's list ------------------------------------------------------------------------------------------------

def _topk(logits: Tensor, inv_T: float, k: int) -> tuple[Tensor, Tensor]:
    dev = _on_gpu(logits)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids = torch.empty(n, k, dtype=torch.int64, device=dev)
    logp = torch.empty(n, k, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.call("octo_topk", _p(z), z.stride(0), _DT[z.dtype], n, V, inv_T, k, _p(ids), _p(logp), _stream(z))
    return ids, logp


@torch.library.custom_op("octohead::topk", mutates_args=(), device_types="cuda")
def topk(logits: Tensor, inv_T: float, k: int) -> tuple[Tensor, Tensor]:
    return _topk(logits, inv_T, k)


@topk.register_fake
def _(logits, inv_T, k):
    return (logits.new_empty(logits.shape[0], k, dtype=torch.int64),
            logits.new_empty(logits.shape[0], k, dtype=torch.float32))


def head_topk(logits: Tensor, temperature: float, k: int) -> tuple[Tensor, Tensor]:
    """(ids [n, k] int64, logp [n, k] fp32): the k largest logits of each row of [n, V] and log_softmax(logits /
    temperature) there, by value descending, equal values by token ascending (a NaN counts as the largest, -0 as 0).
    k is at most min(V, 256). Not differentiable: it is a teacher's answer."""
    if logits.dim() != 2:
        raise ValueError(f"octohead: logits must be [n, V], got {tuple(logits.shape)}")
    inv_T = _inv_T(temperature)
    if not 1 <= k <= min(logits.shape[1], _lib.LIST_MAX):
        raise ValueError(f"octohead: a list of {k} from {logits.shape[1]} logits (at most {_lib.LIST_MAX})")
    logits = logits.detach()
    return topk(logits, inv_T, k) if torch.compiler.is_compiling() else _topk(logits, inv_T, k)


# ---- the divergence over materialised logits -----------------------------------------------------------------------------

@torch.library.custom_op("octohead::distill_columns_fwd", mutates_args=(), device_types="cuda")
def distill_columns_fwd(logits: Tensor, ids: Tensor, teacher: Tensor, inv_T: float,
                        raw: bool) -> tuple[Tensor, Tensor, Tensor]:
    """(kl [n], state [n, 4], q [n, K]), the last two for distill_columns_bwd."""
    dev = _on_gpu(logits, ids, teacher)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids, teacher = _lists(ids, teacher, n)
    K = ids.shape[1]
    kl = torch.empty(n, dtype=torch.float32, device=dev)
    state = torch.empty(n, 4, dtype=torch.float32, device=dev)
    q = torch.empty(n, K, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.call("octo_distill_columns_fwd", _p(z), z.stride(0), _DT[z.dtype], _p(ids), _p(teacher), n, V, K, inv_T,
                  _lib.LIST_RAW if raw else 0, _p(kl), _p(state), _p(q), _stream(z))
    return kl, state, q


@distill_columns_fwd.register_fake
def _(logits, ids, teacher, inv_T, raw):
    f = lambda *s: logits.new_empty(*s, dtype=torch.float32)  # noqa: E731
    return f(logits.shape[0]), f(logits.shape[0], 4), f(*ids.shape)


@torch.library.custom_op("octohead::distill_columns_bwd", mutates_args=(), device_types="cuda")
def distill_columns_bwd(logits: Tensor, ids: Tensor, q: Tensor, inv_T: float, state: Tensor, g: Tensor) -> Tensor:
    dev = _on_gpu(logits, ids, q, state, g)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids, q = _lists(ids, q, n)
    dz = torch.empty(n, V, dtype=z.dtype, device=dev)
    state, g = state.contiguous(), g.float().contiguous()
    with torch.cuda.device(dev):
        _lib.call("octo_distill_columns_bwd", _p(z), z.stride(0), _DT[z.dtype], _p(ids), _p(q), n, V, ids.shape[1],
                  inv_T, _p(state), _p(g), _p(dz), V, _stream(z))
    return dz


@distill_columns_bwd.register_fake
def _(logits, ids, q, inv_T, state, g):
    return logits.new_empty(logits.shape)


def _columns_setup(ctx, inputs, output):
    logits, ids, _teacher, inv_T, _raw = inputs
    ctx.save_for_backward(logits, ids, output[1], output[2])
    ctx.inv_T = inv_T


def _columns_backward(ctx, gkl, _gstate, _gq):
    logits, ids, state, q = ctx.saved_tensors
    dz = distill_columns_bwd(logits, ids, q, ctx.inv_T, state, gkl) if ctx.needs_input_grad[0] else None
    return dz, None, None, None, None


torch.library.register_autograd("octohead::distill_columns_fwd", _columns_backward, setup_context=_columns_setup)


def distill_columns(logits: Tensor, temperature: float, ids: Tensor, teacher: Tensor, *,
                    normalise: bool = True) -> Tensor:
    """[n] fp32: each row's divergence of softmax(logits / temperature) from its list (the module's formula),
    differentiable in logits (not in the teacher's values). normalise=False: q = exp(teacher) as given, for a list of
    log-probabilities whose missing rest is to carry no weight."""
    if logits.dim() != 2:
        raise ValueError(f"octohead: logits must be [n, V], got {tuple(logits.shape)}")
    return distill_columns_fwd(logits, ids, teacher.detach(), _inv_T(temperature), not normalise)[0]
