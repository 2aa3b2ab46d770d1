"""Distillation from a teacher's top logits, over libocto_head.so.

    head_topk                          the teacher's list: the k largest logits of a row and their log-probabilities
    octohead::distill_columns_fwd/bwd  the student's divergence from the lists over materialised logits
    octohead::head_step_distill        the same from hidden rows and the vocabulary weight, with both gradients

A row's list is K slots (ids[r, k], teacher[r, k]): tokens, and the teacher's logits or log-probabilities of them, as
head_topk gives them. A slot whose id lies outside [0, V) or whose teacher value is -inf is empty (shorter lists), and
the same token may stand in several slots. With q the softmax of the teacher's values over a row's slots and p =
softmax(z / T) the student's distribution over the whole vocabulary,

    kl_r = sum_k q_k (log q_k - log p_ids[k])                             (a row without a slot: 0)
    dL/dz_v = g_r (Q p_v - sum of q_k over the slots of v) / T,  Q = sum q,  g_r = dL/dkl_r.

HIP tensors only; all work is queued on the current stream of the tensors' device, nothing synchronises with the host.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib, head_op
from .embed_op import _call_on, _float_rows, _ids, _ld, _on_gpu
from .head_op import (_DT, Post, _dtype_code, _empty, _gather_flag, _index, _later_bytes, _p, _rows2d,
                      _workspace, _zeros, later_grad_w, scaled)


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
    inv_T = 1.0 / float(temperature)
    if not 0.0 < inv_T < 1e38:
        raise ValueError(f"temperature {temperature} lies outside fp32's range")
    return inv_T


# ---- the teacher's list ----------------------------------------------------------------------------------------------

def _topk(logits: Tensor, inv_T: float, k: int) -> tuple[Tensor, Tensor]:
    dev = _on_gpu(logits)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids = torch.empty(n, k, dtype=torch.int64, device=dev)
    logp = torch.empty(n, k, dtype=torch.float32, device=dev)
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_topk_workspace_bytes", n, V, _DT[z.dtype], k, ctypes.byref(nbytes))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
    _call_on(dev, "octo_topk", _p(z), _ld(z), _DT[z.dtype], n, V, inv_T, k, _p(ids), _p(logp), _p(ws), nbytes.value)
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


# ---- the divergence over materialised logits -------------------------------------------------------------------------

def _columns_fwd(logits: Tensor, ids: Tensor, teacher: Tensor, inv_T: float, raw: bool) -> tuple[Tensor, ...]:
    """(kl, state, q, and the logits and ids as the kernels read them)."""
    dev = _on_gpu(logits, ids, teacher)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids, teacher = _lists(ids, teacher, n)
    K = ids.shape[1]
    kl = torch.empty(n, dtype=torch.float32, device=dev)
    state = torch.empty(n, 4, dtype=torch.float32, device=dev)
    q = torch.empty(n, K, dtype=torch.float32, device=dev)
    _call_on(dev, "octo_distill_columns_fwd", _p(z), _ld(z), _DT[z.dtype], _p(ids), _p(teacher), n, V, K, inv_T,
             _lib.LIST_RAW if raw else 0, _p(kl), _p(state), _p(q))
    return kl, state, q, z, ids


@torch.library.custom_op("octohead::distill_columns_fwd", mutates_args=(), device_types="cuda")
def distill_columns_fwd(logits: Tensor, ids: Tensor, teacher: Tensor, inv_T: float,
                        raw: bool) -> tuple[Tensor, Tensor, Tensor]:
    """(kl [n], state [n, 4], q [n, K]), the last two for distill_columns_bwd."""
    return _columns_fwd(logits, ids, teacher, inv_T, raw)[:3]


@distill_columns_fwd.register_fake
def _(logits, ids, teacher, inv_T, raw):
    f = lambda *s: logits.new_empty(*s, dtype=torch.float32)  # noqa: E731
    return f(logits.shape[0]), f(logits.shape[0], 4), f(*ids.shape)


def _columns_bwd(logits: Tensor, ids: Tensor, q: Tensor, inv_T: float, state: Tensor, g: Tensor) -> Tensor:
    dev = _on_gpu(logits, ids, q, state, g)
    z = _float_rows(logits, "logits")
    n, V = z.shape
    ids, q = _lists(ids, q, n)
    return _columns_grad(z, ids, q, inv_T, state.contiguous(), g)


def _columns_grad(z: Tensor, ids: Tensor, q: Tensor, inv_T: float, state: Tensor, g: Tensor) -> Tensor:
    """Of a forward's own tensors, not looked at again."""
    n, V = z.shape
    dz = torch.empty(n, V, dtype=z.dtype, device=z.device)
    g = g.float().contiguous()
    _call_on(z.device, "octo_distill_columns_bwd", _p(z), _ld(z), _DT[z.dtype], _p(ids), _p(q), n, V, ids.shape[1],
             inv_T, _p(state), _p(g), _p(dz), V)
    return dz


@torch.library.custom_op("octohead::distill_columns_bwd", mutates_args=(), device_types="cuda")
def distill_columns_bwd(logits: Tensor, ids: Tensor, q: Tensor, inv_T: float, state: Tensor, g: Tensor) -> Tensor:
    return _columns_bwd(logits, ids, q, inv_T, state, g)


@distill_columns_bwd.register_fake
def _(logits, ids, q, inv_T, state, g):
    return logits.new_empty(logits.shape)


def _columns_setup(ctx, inputs, output):
    logits, ids, _teacher, inv_T, _raw = inputs
    ctx.save_for_backward(logits, ids, output[1], output[2])
    ctx.inv_T = inv_T
    ctx.set_materialize_grads(False)


def _only(name: str, *others: Optional[Tensor]) -> None:
    """Gradients of an op's outputs beside the differentiable one: none may have come in."""
    if any(g is not None for g in others):
        raise RuntimeError(f"octohead: of this op's outputs only {name} is differentiable")


def _columns_backward(ctx, gkl, gstate, gq):
    _only("kl", gstate, gq)
    logits, ids, state, q = ctx.saved_tensors
    dz = distill_columns_bwd(logits, ids, q, ctx.inv_T, state, gkl) \
        if ctx.needs_input_grad[0] and gkl is not None else None
    return dz, None, None, None, None


torch.library.register_autograd("octohead::distill_columns_fwd", _columns_backward, setup_context=_columns_setup)


class _Columns(torch.autograd.Function):
    """distill_columns_fwd and its backward outside a trace, without the registered ops' own bookkeeping on the host (57
    rows of 128,257: 98 us a forward and backward through the ops). With create_graph the backward is the registered op,
    which ties the gradient to the logits it depends on and refuses its derivative."""

    @staticmethod
    def forward(ctx, *args):
        kl, state, q, z, ids = _columns_fwd(*args)
        ctx.save_for_backward(z, ids, state, q)
        ctx.inv_T = args[3]
        return kl

    @staticmethod
    def backward(ctx, gkl):
        z, ids, state, q = ctx.saved_tensors
        if torch.is_grad_enabled():
            return (distill_columns_bwd(z, ids, q, ctx.inv_T, state, gkl),) + (None,) * 4
        return (_columns_grad(z, ids, q, ctx.inv_T, state, gkl),) + (None,) * 4


def distill_columns(logits: Tensor, temperature: float, ids: Tensor, teacher: Tensor, *,
                    normalise: bool = True) -> Tensor:
    """[n] fp32: each row's divergence of softmax(logits / temperature) from its list (the module's formula),
    differentiable in logits (not in the teacher's values). normalise=False: q = exp(teacher) as given, for a list of
    log-probabilities whose missing rest is to carry no weight."""
    if logits.dim() != 2:
        raise ValueError(f"octohead: logits must be [n, V], got {tuple(logits.shape)}")
    # rows the kernels can read from here on, so that what the backward saves is the tensor that autograd knows
    args = (_float_rows(logits, "logits"), ids, teacher.detach(), _inv_T(temperature), not normalise)
    if torch.compiler.is_compiling():
        return distill_columns_fwd(*args)[0]
    return _Columns.apply(*args) if torch.is_grad_enabled() and logits.requires_grad else _columns_fwd(*args)[0]


# ---- the divergence from hidden rows: loss and gradients in one call -------------------------------------------------

def _apart(x: Tensor) -> Tensor:
    """x with rows that do not overlap (a broadcast one's are one row)."""
    return x if _ld(x) >= x.shape[1] else x.contiguous()


def _step(rows: Tensor, weight: Tensor, w_scale: Optional[Tensor], ids: Tensor, teacher: Tensor,
          row_weight: Optional[Tensor], idx: Optional[Tensor], count: Optional[Tensor], inv_T: float, pre: float,
          post: float, use_tanh: bool, raw: bool, need_rows: bool, need_weight: bool, kept: Optional[Tensor]):
    """(loss, kl, grad_rows, grad_w) of octo_head_step_distill; kept: the buffer that takes grad_w's operands."""
    dev = _on_gpu(rows, weight, w_scale, ids, teacher, row_weight, idx, count)
    rows2, weight2, idx = _apart(_rows2d(rows)), _apart(_rows2d(weight)), _index(idx)
    ids, teacher = _lists(ids, teacher, rows2.shape[0])
    if rows2.shape[1] != weight2.shape[1]:
        raise ValueError(f"octohead: rows of width {rows2.shape[1]} against a weight of width {weight2.shape[1]}")
    if row_weight is not None:
        if row_weight.shape != (rows2.shape[0],):
            raise ValueError(f"octohead: row weights [{rows2.shape[0]}] expected, got {tuple(row_weight.shape)}")
        row_weight = row_weight.float().contiguous()
    if count is not None and (count.dtype != torch.int32 or not count.numel()):
        raise ValueError(f"octohead: a row count of int32 expected (compact_rows), got {count.dtype}")
    if w_scale is not None and (w_scale.dtype != torch.float32 or w_scale.shape != weight2.shape[:1]):
        raise ValueError(f"octohead: one fp32 scale per weight row expected, got {w_scale.dtype} "
                         f"{tuple(w_scale.shape)}")
    w_scale = None if w_scale is None else w_scale.contiguous()
    n_max = idx.numel() if idx is not None else rows2.shape[0]
    V, d = weight2.shape
    K = ids.shape[1]
    every = idx is None and count is None  # every row takes part: each output is written whole
    kl = (torch.empty if every else torch.zeros)(rows2.shape[0], dtype=torch.float32, device=dev)
    loss = (torch.empty if n_max else torch.zeros)((), dtype=torch.float32, device=dev)
    grad_rows = (_empty(rows) if every else _zeros(rows)) if need_rows else rows.new_empty(0)
    grad_w = weight.new_empty(0) if not need_weight or kept is not None else \
        (_zeros(weight) if n_max == 0 else _empty(weight))
    if n_max == 0:
        return loss, kl, grad_rows, grad_w
    code = _dtype_code(weight2)
    if kept is not None:
        nbytes = _lib.later_workspace_bytes(n_max, d, V, code, need_rows)
    elif not (need_rows or need_weight) and code != _lib.FP8E4M3:  # the forward alone, in its own workspace
        nbytes = _lib.workspace_bytes(n_max, d, V, code, _gather_flag(rows2, idx))
    else:
        flags = (_lib.WS_STEP | (0 if need_weight else _lib.WS_NO_GRADW) | (0 if need_rows else _lib.WS_NO_GRADH)
                 | _gather_flag(rows2, idx))
        nbytes = _lib.workspace_bytes(n_max, d, V, code, flags)
        if head_op.STEP_WORKSPACE_BYTES is not None:
            nbytes = int(head_op.STEP_WORKSPACE_BYTES)
    ws = _workspace(nbytes, rows2)
    scratch = torch.empty((2 * K + 3) * n_max, dtype=torch.float32, device=dev)
    dots, q, lse, g = scratch.split([K * n_max, K * n_max, 2 * n_max, n_max])
    lists = _lib.Distill(_p(ids), _p(teacher), _p(row_weight), K, _lib.LIST_RAW if raw else 0, _p(dots), _p(q), _p(g),
                         _p(kl), _p(loss))
    gh = None
    if need_rows:  # compact-order rows; scattered into grad_rows below
        gh = grad_rows if idx is None else torch.empty(n_max, d, dtype=rows2.dtype, device=dev)
    gw = grad_w if need_weight and kept is None else None
    _call_on(dev, "octo_head_step_distill", _p(rows2), rows2.shape[0], _ld(rows2), _dtype_code(rows2),
             _p(weight2), _ld(weight2), code, _p(w_scale), _p(idx), _p(count), n_max, d, V, inv_T, pre, post,
             int(use_tanh), _p(lse), ctypes.byref(lists), _p(gh), d, _dtype_code(rows2) if need_rows else _lib.F32,
             _p(gw), code if gw is not None else _lib.F32, _p(kept), 0 if kept is None else kept.numel(), _p(ws),
             ws.numel())
    if need_rows and idx is not None:
        _call_on(dev, "octo_rows_scatter", _p(gh), d, _dtype_code(gh), _p(idx), _p(count), n_max, d, _p(grad_rows),
                 grad_rows.stride(0), _dtype_code(grad_rows), 0)
    return loss, kl, grad_rows, grad_w


@torch.library.custom_op("octohead::head_step_distill", mutates_args=(), device_types="cuda")
def head_step_distill(rows: Tensor, weight: Tensor, w_scale: Optional[Tensor], ids: Tensor, teacher: Tensor,
                      row_weight: Optional[Tensor], idx: Optional[Tensor], count: Optional[Tensor], inv_T: float,
                      pre: float, post: float, use_tanh: bool, raw: bool, need_rows: bool,
                      need_weight: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(loss, kl [rows], grad_rows [rows, d], grad_weight [V, d]); a gradient not asked for is an empty tensor."""
    return _step(rows, weight, w_scale, ids, teacher, row_weight, idx, count, inv_T, pre, post, use_tanh, raw,
                 need_rows, need_weight, None)


@head_step_distill.register_fake
def _(rows, weight, w_scale, ids, teacher, row_weight, idx, count, inv_T, pre, post, use_tanh, raw, need_rows,
      need_weight):
    return (rows.new_empty((), dtype=torch.float32), rows.new_empty(rows.shape[0], dtype=torch.float32),
            _empty(rows) if need_rows else rows.new_empty(0), _empty(weight) if need_weight else weight.new_empty(0))


class _Final(torch.autograd.Function):
    """A gradient, tied to the tensors it depends on: differentiated, it raises, and is never a silent constant."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("octohead: the gradients of the distillation step have no derivative of their own")


def _final(grads, *of: Optional[Tensor]) -> tuple:
    """The step's gradients as a backward returns them; of: what they depend on."""
    of = [t for t in of if t is not None and t.requires_grad]
    if not (torch.is_grad_enabled() and of):  # no create_graph
        return tuple(grads)
    return tuple(None if t is None else _Final.apply(t.detach(), *of) for t in grads)


def _step_setup(ctx, inputs, output):
    # held as detached aliases, not saved: an offload's pack hook never copies the [V, d] gradient to the host
    ctx.grads = (output[2].detach(), output[3].detach())
    ctx.need, ctx.of = inputs[-2:], inputs[:2]
    ctx.set_materialize_grads(False)


def _step_backward(ctx, gloss, gkl, ggr, ggw):
    _only("loss", gkl, ggr, ggw)
    # into tensors of their own: the op's outputs are its caller's, and a retained graph's second backward reads them
    wanted = [t if ctx.need[k] and ctx.needs_input_grad[k] else None for k, t in enumerate(ctx.grads)]
    out = [None if t is None else torch.zeros_like(t) if gloss is None else scaled(t, gloss) for t in wanted]
    return _final(out, *ctx.of, gloss) + (None,) * 13


torch.library.register_autograd("octohead::head_step_distill", _step_backward, setup_context=_step_setup)


def _step_later(rows: Tensor, weight: Tensor, ids: Tensor, teacher: Tensor, row_weight: Optional[Tensor],
                idx: Optional[Tensor], count: Optional[Tensor], inv_T: float, pre: float, post: float, use_tanh: bool,
                raw: bool, need_rows: bool, nbytes: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(loss, kl, grad_rows, the buffer of nbytes that later_grad_w makes grad_weight of, the row count as the call
    found it)."""
    n_max = idx.numel() if idx is not None else rows.shape[0]
    kept_count = torch.full((1,), n_max, dtype=torch.int32, device=rows.device) if count is None \
        else count.reshape(-1)[:1].to(torch.int32, copy=True)
    kept = _workspace(nbytes, rows)
    loss, kl, grad_rows, _ = _step(rows, weight, None, ids, teacher, row_weight, idx, count, inv_T, pre, post, use_tanh,
                                   raw, need_rows, True, kept)
    return loss, kl, grad_rows, kept, kept_count


def _later_setup(ctx, inputs, output):
    rows, weight, idx = inputs[0], inputs[1], inputs[5]
    ctx.held = (output[2].detach(), output[3].detach(), output[4].detach())
    ctx.sizes = (idx.numel() if idx is not None else rows.shape[0], weight.shape[1], weight.shape[0], weight.dtype)
    ctx.need_rows, ctx.of = inputs[-2], inputs[:2]
    ctx.set_materialize_grads(False)


def _later_backward(ctx, gloss):
    grad_rows, kept, count = ctx.held
    n_max, d, V, dtype = ctx.sizes
    gr = gw = None
    if ctx.need_rows and ctx.needs_input_grad[0]:
        gr = torch.zeros_like(grad_rows) if gloss is None else scaled(grad_rows, gloss)
    if ctx.needs_input_grad[1]:
        gw = torch.zeros(V, d, dtype=dtype, device=kept.device) if gloss is None \
            else later_grad_w(kept, count, gloss, n_max, d, V, dtype, ctx.need_rows)
    return _final((gr, gw), *ctx.of, gloss)


class _Head(torch.autograd.Function):
    """The step outside a trace. It holds its gradients (or operands) for itself, so that the last backward scales them
    where they lie, which ends at once for a loss that is not scaled; a copy reads and writes [V, d] ([151,936, 2560]
    bf16 267 us)."""

    @staticmethod
    def forward(ctx, rows, weight, w_scale, ids, teacher, row_weight, idx, count, xf, need_rows, need_weight, nbytes):
        ctx.later = bool(nbytes)
        if nbytes:
            inputs = (rows, weight, ids, teacher, row_weight, idx, count, *xf, need_rows, nbytes)
            output = _step_later(*inputs)
            _later_setup(ctx, inputs, output)
        else:
            output = _step(rows, weight, w_scale, ids, teacher, row_weight, idx, count, *xf, need_rows, need_weight,
                           None)
            ctx.grads, ctx.need, ctx.of = output[2:], (need_rows, need_weight), (rows, weight)
            ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(output[1])
        return output[0], output[1]

    @staticmethod
    def backward(ctx, gloss, gkl):
        if ctx.later:
            return _later_backward(ctx, gloss) + (None,) * 10
        if ctx.grads is None:
            raise RuntimeError("octohead: the gradients held by the distillation step went with its last backward; "
                               "retain_graph=True keeps them for another")
        if torch._C._autograd._get_current_graph_task_keep_graph() or gloss is None:
            return _step_backward(ctx, gloss, None, None, None)[:2] + (None,) * 10
        held, ctx.grads, ctx.of = ctx.grads, None, ()
        c = gloss.float().contiguous()
        out = [t if ctx.need[k] and ctx.needs_input_grad[k] else None for k, t in enumerate(held)]
        for t in out:
            if t is not None and t.numel():
                _call_on(t.device, "octo_scale_add", _p(t), None, _DT[t.dtype], t.numel(), _p(c), None)
        return (*out,) + (None,) * 10


def fused_distill_head(rows: Tensor, weight: Tensor, ids: Tensor, teacher: Tensor, temperature: float,
                       row_weight: Optional[Tensor] = None, *, normalise: bool = True, post: Post = Post(),
                       idx: Optional[Tensor] = None, count: Optional[Tensor] = None,
                       w_scale: Optional[Tensor] = None) -> tuple[Tensor, Tensor]:
    """(loss, kl): loss = sum over the rows of row_weight x kl (None: 1 each), z = post(rows W^T), and kl [rows] fp32
    detached, from one call that computes the logits once and also the gradients of the loss in rows and weight (each
    when it requires grad and grad mode is on). loss.backward() only scales them or, for a short call, makes the
    weight's from the operands kept, as fused_grpo_head's. ids and teacher are [rows, K], row_weight [rows]. idx, count:
    the rows that take part (ascending, as compact_rows gives them; count on the device); the others' kl and gradients
    are 0. A row of weight 0, or without a slot, adds nothing to the loss, but is computed with: leave rows out by idx,
    and those whose hidden values may be no numbers have to be. bf16, f16, fp32 and fp8 weights (w_scale; no gradient of
    those). The gradients are formed at row_weight's scale and rounded to the operands' type there; in f16 a loss scale
    belongs into row_weight, since loss.backward() multiplies what is rounded already.
    The prefix tree's teacher values depend on the path alone, so a tree's rows are its positions, each once, weighted
    by the tokens that share it. The gradients or operands, and rows and weight by reference, are held from this call
    until the graph goes. The gradients have no derivative of their own: one raises."""
    inv_T = _inv_T(temperature)
    if rows.dim() != 2 or weight.dim() != 2:
        raise ValueError(f"octohead: rows [n, d] and weight [V, d] expected, got {tuple(rows.shape)} and "
                         f"{tuple(weight.shape)}")
    grad_on = torch.is_grad_enabled()
    need_rows, need_weight = grad_on and rows.requires_grad, grad_on and weight.requires_grad
    teacher = teacher.detach()
    row_weight = None if row_weight is None else row_weight.detach()
    xf = (inv_T, float(post.pre), float(post.post), bool(post.tanh), not normalise)
    nbytes = _later_bytes(rows, weight, idx, need_rows, need_weight)
    if not torch.compiler.is_compiling():
        if need_rows or need_weight:
            return _Head.apply(rows, weight, w_scale, ids, teacher, row_weight, idx, count, xf, need_rows, need_weight,
                               nbytes)
        return _step(rows, weight, w_scale, ids, teacher, row_weight, idx, count, *xf, False, False, None)[:2]
    loss, kl, *_ = head_step_distill(rows, weight, w_scale, ids, teacher, row_weight, idx, count, *xf, need_rows,
                                     need_weight)
    return loss, kl.detach()
