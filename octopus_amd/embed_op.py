"""Embedding lookup with scaling and its gradient by sorted tokens, over libocto_head.so.

    octohead::embed_fwd / embed_bwd    scale W[ids], and the gradient in W over the whole vocabulary
    octohead::embed_grad_add           the same gradient added to rows of a gradient that exists already

The other end of the vocabulary matrix that the head multiplies with: a model with tied weights looks its tokens up in
W, and both gradients belong to the one [V, d] tensor. HIP tensors only; all work is queued on the current stream of the
tensors' device, nothing synchronises with the host.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .head_op import _DT, _p, _workspace

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _float_rows(x: Tensor, what: str) -> Tensor:
    """x [rows, d] with contiguous rows."""
    if x.dim() != 2 or not x.shape[1]:
        raise ValueError(f"octohead: {what} must be [rows, d], got {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise NotImplementedError(f"octohead: {what} of dtype {x.dtype} has no HIP kernel")
    return x if x.stride(1) == 1 and (x.shape[0] < 2 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _ld(x: Tensor) -> int:
    """Elements between x's rows; one row's stride may be any number."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _on_gpu(*tensors: Optional[Tensor]) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device != dev):
            raise ValueError(f"octohead: tensors on one HIP device expected, got {dev} and {t.device}")
    return dev


def _call_on(dev: torch.device, name: str, *args) -> None:
    """_lib.call on dev's current stream, its last argument, with dev current. The raw handle, and no entering of a
    device that is current already: the stream's Python object alone takes 10 us in a backward's thread, a tenth of a
    short call."""
    stream = ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(dev.index))
    if torch.cuda.current_device() == dev.index:
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, stream)


def _ids(ids: Tensor) -> Tensor:
    if ids.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
        raise ValueError(f"octohead: ids must be integers, got {ids.dtype}")
    return ids.to(torch.int64).contiguous()


def _fwd(weight: Tensor, ids: Tensor, scale: float) -> Tensor:
    dev = _on_gpu(weight, ids)
    w = _float_rows(weight, "weight")
    flat = _ids(ids).reshape(-1)
    V, d = w.shape
    if V == 0:
        raise ValueError("octohead: an empty vocabulary")
    out = torch.empty(*ids.shape, d, dtype=w.dtype, device=dev)
    _call_on(dev, "octo_embed_fwd", _p(w), _ld(w), _DT[w.dtype], V, d, _p(flat), flat.numel(), float(scale),
             _p(out), d)
    return out


def _bwd(into: Tensor, grad: Tensor, ids: Tensor, scale: float, padding_idx: int, accumulate: bool) -> None:
    dev = _on_gpu(into, grad, ids)
    V, d = into.shape
    flat = _ids(ids).reshape(-1)
    n = flat.numel()
    if tuple(grad.shape) != (*ids.shape, d):
        raise ValueError(f"octohead: gradient {tuple(grad.shape)} for ids {tuple(ids.shape)} of width {d}")
    g = _float_rows(grad.reshape(n, d), "gradient")
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_embed_bwd_workspace_bytes", n, V, d, ctypes.byref(nbytes))
    ws = _workspace(nbytes.value, into)
    _call_on(dev, "octo_embed_bwd", _p(g), _ld(g), _DT[g.dtype], _p(flat), n, V, d, padding_idx, float(scale),
             _p(into), _ld(into), _DT[into.dtype], int(accumulate), _p(ws), ws.numel())


@torch.library.custom_op("octohead::embed_fwd", mutates_args=(), device_types="cuda")
def embed_fwd(weight: Tensor, ids: Tensor, scale: float, padding_idx: int) -> Tensor:
    return _fwd(weight, ids, scale)


@embed_fwd.register_fake
def _(weight, ids, scale, padding_idx):
    return weight.new_empty(*ids.shape, weight.shape[1])


def _gradient(grad: Tensor, ids: Tensor, V: int, scale: float, padding_idx: int, dtype: torch.dtype) -> Tensor:
    if dtype not in _FLOATS:
        raise NotImplementedError(f"octohead: a gradient of dtype {dtype} has no HIP kernel")
    if V <= 0 or grad.dim() < 1 or not grad.shape[-1]:
        raise ValueError(f"octohead: gradient {tuple(grad.shape)} over {V} entries")
    out = torch.empty(V, grad.shape[-1], dtype=dtype, device=grad.device)
    _bwd(out, grad, ids, scale, padding_idx, False)
    return out


@torch.library.custom_op("octohead::embed_bwd", mutates_args=(), device_types="cuda")
def _embed_bwd(grad: Tensor, ids: Tensor, V: int, scale: float, padding_idx: int, dtype: torch.dtype) -> Tensor:
    return _gradient(grad, ids, V, scale, padding_idx, dtype)


@_embed_bwd.register_fake
def _(grad, ids, V, scale, padding_idx, dtype):
    return grad.new_empty(V, grad.shape[-1], dtype=dtype)


@torch.library.custom_op("octohead::embed_grad_add", mutates_args=("into",), device_types="cuda")
def _embed_grad_add(into: Tensor, grad: Tensor, ids: Tensor, scale: float, padding_idx: int) -> None:
    if _float_rows(into, "gradient to add to") is not into:
        raise ValueError("octohead: the gradient to add to needs contiguous rows")
    _bwd(into, grad, ids, scale, padding_idx, True)


@_embed_grad_add.register_fake
def _(into, grad, ids, scale, padding_idx):
    return None


def _op(op, plain):
    """The registered op inside a trace, else the call behind it."""
    return op if torch.compiler.is_compiling() else plain


def _setup(ctx, inputs, output):
    weight, ids, scale, padding_idx = inputs
    ctx.save_for_backward(ids)
    ctx.params = (weight.shape[0], scale, padding_idx, weight.dtype)


def _backward(ctx, gout, gradient=_embed_bwd):
    """The registered op's own backward calls the registered gradient: a tracer runs it on tensors without data, and
    with create_graph its result depends on gout, whose derivative is refused and not left out."""
    (ids,) = ctx.saved_tensors
    V, scale, padding_idx, dtype = ctx.params
    gw = gradient(gout, ids, V, scale, padding_idx, dtype) if ctx.needs_input_grad[0] else None
    return gw, None, None, None


torch.library.register_autograd("octohead::embed_fwd", _backward, setup_context=_setup)


class _Embed(torch.autograd.Function):
    """embed_fwd outside a trace: the registered op's own bookkeeping takes longer on the host than the kernel does for
    a step's tokens (16 tokens: 31 us a call through the op, 13 through the library)."""

    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        _setup(ctx, (weight, ids, scale, padding_idx), None)
        return _fwd(weight, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        return _backward(ctx, gout, _gradient)


def _padding(padding_idx: Optional[int], V: int) -> int:
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise ValueError(f"octohead: padding_idx {padding_idx} outside a vocabulary of {V}")
    return padding_idx % V


def embed_rows(weight: Tensor, ids: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """[*ids.shape, d] in weight's dtype: scale x weight[ids], the product formed in fp32 and rounded once; zeros for an
    id outside [0, V) (a packed stream's filling). Differentiable in weight: embed_bwd's gradient, dense over the
    vocabulary. padding_idx: an entry that is looked up and gets no gradient."""
    if weight.dim() != 2:
        raise ValueError(f"octohead: weight must be [V, d], got {tuple(weight.shape)}")
    pad = _padding(padding_idx, weight.shape[0])
    if torch.compiler.is_compiling():
        return embed_fwd(weight, ids, float(scale), pad)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embed.apply(weight, ids, float(scale), pad)
    return _fwd(weight, ids, scale)


def embed_bwd(grad: Tensor, ids: Tensor, V: int, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> Tensor:
    """[V, d] in dtype (None: grad's): scale x the sum of grad [*ids.shape, d] over the tokens of each entry, zeros for
    an entry without one. Summed in fp32 in an order that the ids alone decide (equal calls, equal bits), rounded once.
    ids outside [0, V) and padding_idx are left out."""
    return _op(_embed_bwd, _gradient)(grad, ids, V, float(scale), _padding(padding_idx, V), dtype or grad.dtype)


def embed_grad_add_(into: Tensor, grad: Tensor, ids: Tensor, scale: float = 1.0,
                    padding_idx: Optional[int] = None) -> Tensor:
    """embed_bwd's sums added in place to the rows of into [V, d] that the tokens name, each added in fp32 and rounded
    once; the other rows are neither read nor written. For tied weights: into is the gradient the head has left, so that
    no second [V, d] tensor is written, read and added. Returns into."""
    if into.dim() != 2:
        raise ValueError(f"octohead: the gradient to add to must be [V, d], got {tuple(into.shape)}")
    _embed_grad_add(into, grad, ids, float(scale), _padding(padding_idx, into.shape[0]))
    return into
