"""8-bit integers at the vocabulary's end, over libocto_head.so: rows held in 8 bits, and the head's logits from them.

    octohead::quantise_rows / widen_rows       rows as int8 with fp32 scales, and back
    octohead::head_logits_i8 / head_grads_i8   rows W^T in 8-bit integers, a scale for each row of both; its gradients
    checkpoint8                                a checkpoint that holds its inputs in 8 bits

Of a row, or of each group of 32 to 256 of its values, with a the largest magnitude: scale = a times 1/127, both in
fp32, q the exact quotient x / scale to the nearest integer (ties to even). A group below 2^-119 is held as zeros, one
with a NaN or an infinity as NaN. int8 rows start on 16-byte boundaries, zeros between them (quantise_rows gives them
so).

The logits are x_scale w_scale sum_k xq wq, the sum exact. Their gradients go straight through the rounding: in the rows
g (w_scale wq), in the weight g^T (x_scale xq), so that what is held for them is the 8-bit rows that the product read
and not the rows. HIP tensors only; all work is queued on the current stream of the tensors' device, nothing
synchronises with the host.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from . import _lib
from .embed_op import _FLOATS, _call_on, _float_rows, _ld, _on_gpu
from .head_op import _DT, _p, _workspace

GROUPS = (0, 32, 64, 128, 256)
_F32_GRADS_MAX = 1 << 20  # rows and columns of fp32 gradients: three parts of each within the products' 32-bit offsets


def _ld8(d: int) -> int:
    return -(-d // 16) * 16


def _groups(d: int, group: int) -> int:
    if group not in GROUPS:
        raise ValueError(f"octohead: groups of 32, 64, 128 or 256 values, or 0 for a scale a row, got {group}")
    return -(-d // group) if group else 1


def _scale_shape(shape, group: int) -> tuple:
    return (*shape[:-1], _groups(shape[-1], group)) if group else tuple(shape[:-1])


def _rows_of(x: Tensor, what: str) -> Tensor:
    """[*, d] as [rows, d] that the kernels can read."""
    if x.dim() == 2:
        return _float_rows(x, what)
    if x.dim() < 1 or not x.shape[-1]:
        raise ValueError(f"octohead: {what} must be [*, d], got {tuple(x.shape)}")
    return _float_rows(x.reshape(-1, x.shape[-1]), what)


def _rows8(q: Tensor) -> Tensor:
    """q [*, d] int8 as [rows, d], rows on 16-byte boundaries and readable up to the next; a copy where they are not."""
    if q.dtype != torch.int8 or q.dim() < 1 or not q.shape[-1]:
        raise ValueError(f"octohead: int8 rows [*, d] expected, got {q.dtype} {tuple(q.shape)}")
    if q.dim() != 2:
        q = q.reshape(-1, q.shape[-1])
    n, d = q.shape
    whole = _ld8(d)
    ld, one = q.stride()
    if n < 2:
        ld = whole
    if one == 1 and ld % 16 == 0 and whole <= ld <= 262144 and q.data_ptr() % 16 == 0 and \
            (ld == d or q.untyped_storage().nbytes() >= q.storage_offset() + max(n - 1, 0) * ld + whole):
        return q
    out = torch.zeros(n, whole, dtype=torch.int8, device=q.device)[:, :d]
    return out.copy_(q)


def _ldq(q: Tensor) -> int:
    return q.stride(0) if q.shape[0] > 1 else _ld8(q.shape[1])


def _scales(scale: Tensor, shape, what: str) -> Tensor:
    if scale.dtype != torch.float32 or scale.shape != shape:
        raise ValueError(f"octohead: {what} of fp32 {tuple(shape)} expected, got {scale.dtype} {tuple(scale.shape)}")
    return scale.contiguous()


# ---- rows held in 8 bits ---------------------------------------------------------------------------------------------

def _quantise(x: Tensor, group: int) -> tuple[Tensor, Tensor]:
    dev = _on_gpu(x)
    rows = _rows_of(x, "rows")
    n, d = rows.shape
    q = torch.empty(*x.shape[:-1], _ld8(d), dtype=torch.int8, device=dev)
    scale = torch.empty(_scale_shape(x.shape, group), dtype=torch.float32, device=dev)
    _call_on(dev, "octo_quantise_i8_rows", _p(rows), _ld(rows), _DT[rows.dtype], n, d, group, _p(q), _ld8(d), _p(scale))
    return q if d % 16 == 0 else q[..., :d], scale


@torch.library.custom_op("octohead::quantise_rows", mutates_args=(), device_types="cuda")
def _quantise_op(x: Tensor, group: int) -> tuple[Tensor, Tensor]:
    return _quantise(x, group)


@_quantise_op.register_fake
def _(x, group):
    d = x.shape[-1]
    return (x.new_empty(*x.shape[:-1], _ld8(d), dtype=torch.int8)[..., :d],
            x.new_empty(_scale_shape(x.shape, group), dtype=torch.float32))


def quantise_rows(x: Tensor, group: int = 0) -> tuple[Tensor, Tensor]:
    """(q int8 [*, d], scale fp32 [*] or, with a group, [*, ceil(d / group)]) of x [*, d] in bf16, f16 or fp32 (the
    module's format). Not differentiable."""
    _groups(1, group)
    return _quantise_op(x.detach(), group) if torch.compiler.is_compiling() else _quantise(x, group)


def _widen(q: Tensor, scale: Tensor, dtype: torch.dtype, group: int) -> Tensor:
    dev = _on_gpu(q, scale)
    if dtype not in _FLOATS:
        raise NotImplementedError(f"octohead: rows of dtype {dtype} have no HIP kernel")
    rows = _rows8(q)
    n, d = rows.shape
    scale = _scales(scale, _scale_shape(q.shape, group), "scales")
    out = torch.empty(q.shape, dtype=dtype, device=dev)
    _call_on(dev, "octo_widen_i8_rows", _p(rows), _ldq(rows), _p(scale), n, d, group, _p(out), d, _DT[dtype])
    return out


@torch.library.custom_op("octohead::widen_rows", mutates_args=(), device_types="cuda")
def _widen_op(q: Tensor, scale: Tensor, dtype: torch.dtype, group: int) -> Tensor:
    return _widen(q, scale, dtype, group)


@_widen_op.register_fake
def _(q, scale, dtype, group):
    return q.new_empty(q.shape, dtype=dtype)


def widen_rows(q: Tensor, scale: Tensor, dtype: torch.dtype, group: int = 0) -> Tensor:
    """[*, d] in dtype: q times its scales in fp32, rounded to dtype. What quantise_rows(x, group) took comes back
    within half a step of its scale and those roundings. Not differentiable."""
    _groups(1, group)
    return _widen_op(q, scale, dtype, group) if torch.compiler.is_compiling() else _widen(q, scale, dtype, group)


def _holds(x, group: int) -> bool:
    """Whether x is held in 8 bits: where the bytes of a row, padded, with its scales, are fewer than x's own (16-bit
    rows from d 11 on, but for 17 and 18). A tensor that is expanded takes less as it is; a parameter is there anyway,
    and fn may read more of another class of tensors than its values."""
    if type(x) is not Tensor or not (x.requires_grad and torch.is_grad_enabled() and x.is_cuda and
                                     x.dtype in _FLOATS and x.dim() > 0 and x.shape[-1] > 0) or \
            any(step == 0 and size > 1 for size, step in zip(x.shape, x.stride())):
        return False
    d = x.shape[-1]
    return _ld8(d) + 4 * _groups(d, group) < d * x.element_size()


def checkpoint8(fn, *xs, group: int = 128):
    """fn(*xs), recomputed in the backward (torch.utils.checkpoint, not reentrant) from inputs that are held in 8 bits
    in between: those of bf16, f16 or fp32 on a HIP device that require a gradient, are plain tensors (no parameters nor
    other subclasses) and take fewer bytes so (not the narrowest rows, nor a tensor that is expanded). The forward sees
    them as they are, the recompute what their 8 bits stand for, so what fn saves for its gradients is off by the
    rounding (half of 1/127 of a group's largest value). They have to be finite: a group with a NaN or an infinity (-inf
    in a bias that is learnt) is NaN in the recompute. Other arguments (masks, positions, parameters, None) are kept by
    reference; changed in place before the backward, it raises, as an ordinary checkpoint does."""
    _groups(1, group)
    live = list(xs)
    dtypes = [x.dtype if _holds(x, group) else None for x in xs]

    def run(*kept):
        if live:  # the forward itself
            args = live[:]
            live.clear()
        else:
            rest = iter(kept)
            args = [next(rest) if t is None else widen_rows(next(rest), next(rest), t, group).requires_grad_(True)
                    for t in dtypes]
        return fn(*args)

    # All that is kept, 8-bit rows and scales too, goes through the checkpoint's own arguments: it watches them for
    # changes in place, finds in them the devices whose random numbers fn draws, and shows them to saved tensors' hooks.
    kept = [y for x, t in zip(xs, dtypes) for y in ((x,) if t is None else quantise_rows(x, group))]
    return checkpoint(run, *kept, use_reentrant=False)


# ---- the head's logits -----------------------------------------------------------------------------------------------

def _weights(rows: Tensor, wq: Tensor, w_scale: Tensor, weight: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    if wq.dim() != 2:
        raise ValueError(f"octohead: int8 weights [V, d] expected, got {tuple(wq.shape)}")
    V, d = wq.shape
    if rows.dim() < 1 or rows.shape[-1] != d:
        raise ValueError(f"octohead: rows {tuple(rows.shape)} against weights of width {d}")
    if weight is not None and tuple(weight.shape) != (V, d):
        raise ValueError(f"octohead: weight {tuple(weight.shape)} for int8 weights {tuple(wq.shape)}")
    return _rows8(wq), _scales(w_scale, (V,), "one scale per weight row")


def _logits(rows: Tensor, wq: Tensor, w_scale: Tensor, weight: Optional[Tensor],
            out_dtype: torch.dtype) -> tuple[Tensor, ...]:
    """(logits, xq, x_scale, and the weights as the kernels read them)."""
    dev = _on_gpu(rows, wq, w_scale, weight)
    if out_dtype not in _FLOATS:
        raise NotImplementedError(f"octohead: logits of dtype {out_dtype} have no HIP kernel")
    x = _rows_of(rows, "rows")
    w8, ws = _weights(rows, wq, w_scale, weight)
    n, d = x.shape
    V = w8.shape[0]
    xq = torch.empty(n, _ld8(d), dtype=torch.int8, device=dev)
    xs = torch.empty(n, dtype=torch.float32, device=dev)
    z = torch.empty(*rows.shape[:-1], V, dtype=out_dtype, device=dev)
    _call_on(dev, "octo_head_logits_i8", _p(x), _ld(x), _DT[x.dtype], _p(w8), _ldq(w8), _p(ws), n, d, V, _p(xq),
             _ld8(d), _p(xs), _p(z), V, _DT[out_dtype])
    return z, xq[:, :d], xs, w8, ws


def _grads(g: Tensor, xq: Tensor, xs: Tensor, w8: Tensor, ws: Tensor, rows_dtype: torch.dtype, w_dtype: torch.dtype,
           need_rows: bool, need_w: bool) -> tuple[Optional[Tensor], Optional[Tensor]]:
    """(grad_rows [n, d], grad_w [V, d]) of g [*, V]."""
    dev = _on_gpu(g, xq, xs, w8, ws)
    V, d = w8.shape
    n = xq.shape[0]
    if g.shape[-1] != V or g.numel() != n * V:
        raise ValueError(f"octohead: gradient {tuple(g.shape)} for {n} rows of {V} logits")
    g = _rows_of(g, "gradient")
    gr = torch.empty(n, d, dtype=rows_dtype, device=dev) if need_rows else None
    gw = (torch.empty if n else torch.zeros)(V, d, dtype=w_dtype, device=dev) if need_w else None
    if n == 0 or not (need_rows or need_w):
        return gr, gw
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_head_grads_i8_workspace_bytes", _p(g), _ld(g), _DT[g.dtype], n, d, V, int(need_rows), int(need_w),
              ctypes.byref(nbytes))
    work = _workspace(nbytes.value, g)
    _call_on(dev, "octo_head_grads_i8", _p(g), _ld(g), _DT[g.dtype], _p(xq), _ldq(xq), _p(xs), _p(w8), _ldq(w8),
             _p(ws), n, d, V, _p(gr), d, _DT[rows_dtype], _p(gw), d, _DT[w_dtype], _p(work), work.numel())
    return gr, gw


@torch.library.custom_op("octohead::head_logits_i8", mutates_args=(), device_types="cuda")
def head_logits_i8(rows: Tensor, wq: Tensor, w_scale: Tensor, weight: Optional[Tensor],
                   out_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    """(logits [*, V], xq [n, d], x_scale [n]), the last two for head_grads_i8."""
    return _logits(rows, wq, w_scale, weight, out_dtype)[:3]


@head_logits_i8.register_fake
def _(rows, wq, w_scale, weight, out_dtype):
    n, d = rows.numel() // rows.shape[-1], rows.shape[-1]
    return (rows.new_empty(*rows.shape[:-1], wq.shape[0], dtype=out_dtype),
            rows.new_empty(n, _ld8(d), dtype=torch.int8)[:, :d], rows.new_empty(n, dtype=torch.float32))


@torch.library.custom_op("octohead::head_grads_i8", mutates_args=(), device_types="cuda")
def head_grads_i8(g: Tensor, xq: Tensor, x_scale: Tensor, wq: Tensor, w_scale: Tensor, rows_dtype: torch.dtype,
                  w_dtype: torch.dtype, need_rows: bool, need_w: bool) -> tuple[Tensor, Tensor]:
    """(grad_rows [n, d], grad_weight [V, d]); one not asked for is an empty tensor."""
    gr, gw = _grads(g, _rows8(xq), x_scale.contiguous(), _rows8(wq), w_scale.contiguous(), rows_dtype, w_dtype,
                    need_rows, need_w)
    return (g.new_empty(0, dtype=rows_dtype) if gr is None else gr,
            g.new_empty(0, dtype=w_dtype) if gw is None else gw)


@head_grads_i8.register_fake
def _(g, xq, x_scale, wq, w_scale, rows_dtype, w_dtype, need_rows, need_w):
    return (g.new_empty(xq.shape if need_rows else (0,), dtype=rows_dtype),
            g.new_empty(wq.shape if need_w else (0,), dtype=w_dtype))


def _setup(ctx, inputs, output):
    rows, wq, w_scale, weight, _ = inputs
    ctx.save_for_backward(output[1], output[2], wq, w_scale)
    ctx.like = (rows.shape, rows.dtype, None if weight is None else weight.dtype)
    ctx.set_materialize_grads(False)


def _backward(ctx, g, *others):
    """The registered op's own backward calls the registered gradients: a tracer runs it on tensors without data, and
    with create_graph its result depends on g, whose derivative is refused and not left out."""
    if any(o is not None for o in others):
        raise RuntimeError("octohead: of this op's outputs only the logits are differentiable")
    need_rows, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
    if g is None or not (need_rows or need_w):
        return (None,) * 5
    shape, dtype, w_dtype = ctx.like
    gr, gw = head_grads_i8(g, *ctx.saved_tensors, dtype, w_dtype or dtype, need_rows, need_w)
    return gr.view(shape) if need_rows else None, None, None, gw if need_w else None, None


torch.library.register_autograd("octohead::head_logits_i8", _backward, setup_context=_setup)


def _version(t: Tensor) -> Optional[int]:
    return None if t.is_inference() else t._version


class _Head8(torch.autograd.Function):
    """head_logits_i8 and its backward outside a trace, without the registered ops' own bookkeeping on the host. With
    create_graph the backward is the registered op, which refuses its derivative."""

    @staticmethod
    def forward(ctx, rows, wq, w_scale, weight, out_dtype):
        z, xq, xs, w8, ws = _logits(rows, wq, w_scale, weight, out_dtype)
        ctx.save_for_backward(xq, xs)
        # the weights by reference, not saved: an offload's pack hook never copies the [V, d] bytes to the host
        ctx.weights, ctx.watched = (w8, ws), [(t, _version(t)) for t in (wq, w_scale)]
        ctx.like = (rows.shape, rows.dtype, None if weight is None else weight.dtype)
        return z

    @staticmethod
    def backward(ctx, g):
        need_rows, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        for t, version in ctx.watched:
            if _version(t) != version:
                raise RuntimeError("octohead: the 8-bit weights were changed in place between the logits and their "
                                   "backward")
        shape, dtype, w_dtype = ctx.like
        call = head_grads_i8 if torch.is_grad_enabled() else _grads
        xq, xs = ctx.saved_tensors
        xq = _rows8(xq)  # as saved, or as a hook gave them back: without the bytes between the rows
        gr, gw = call(g, xq, xs, *ctx.weights, dtype, w_dtype or dtype, need_rows, need_w)
        return gr.view(shape) if need_rows else None, None, None, gw if need_w else None, None


def int8_head(rows: Tensor, wq: Tensor, w_scale: Tensor, *, weight: Optional[Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """Logits [*, V] in out_dtype (None: rows') of rows [*, d] in bf16, f16 or fp32 against a vocabulary matrix in 8
    bits, (wq, w_scale) = quantise_rows(weight): each row quantised here, the product exact in 32-bit integers, scaled
    in fp32 and rounded to the logits' type. The rows' gradient is that of the weights' 8-bit values. weight: the [V, d]
    parameter that wq was made of, which gets the gradient straight through the rounding; its values are not read, and
    wq is made again when it has changed. For 16-bit logits the 8-bit operands times their scales are rounded to the
    logits' type before the gradients' products, which leaves them 2.4e-3 (bf16) or 2.9e-4 (f16) from 64 bits; those of
    fp32 logits are within 1e-6. Between the two passes the rows are held in 8 bits, and wq and w_scale by reference
    (changed in place, the backward raises). wq and w_scale get no gradient; the gradients have no derivative of their
    own and the logits none in forward mode (one raises)."""
    out_dtype = out_dtype or rows.dtype
    train = torch.is_grad_enabled() and (rows.requires_grad or weight is not None and weight.requires_grad)
    if train and out_dtype == torch.float32 and wq.dim() == 2:
        V, d = wq.shape
        n = rows.numel() // max(d, 1)
        if max(n, V) > _F32_GRADS_MAX:
            raise ValueError(f"octohead: fp32 logits [{n}, {V}] have gradients up to {_F32_GRADS_MAX} rows and columns")
    if torch.compiler.is_compiling():
        return head_logits_i8(rows, wq, w_scale, weight, out_dtype)[0]
    if forward_ad._current_level >= 0 and \
            any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (rows, w_scale, weight)):
        raise NotImplementedError("octohead: the 8-bit head's logits have no derivative in forward mode")
    if train:
        return _Head8.apply(rows, wq, w_scale, weight, out_dtype)
    return _logits(rows, wq, w_scale, weight, out_dtype)[0]
