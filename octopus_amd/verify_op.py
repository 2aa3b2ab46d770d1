"""Verification of drafted tokens against the target's probabilities, over libocto_head.so.

    octohead::verify_drafts   the tokens a sequence answers with, from given random numbers, and their log-probabilities

With p_i = softmax(target logits_i / T), q_i = softmax(draft logits_i / T) and u given numbers in [0, 1):

    draft i is accepted when u_i q_i(x_i) < p_i(x_i); the first that is not ends the drafts at a
    the next token is the lowest v with sum_{w <= v} r_w > u_K sum r, r = max(p_a - q_a, 0), p_a behind the last draft

so the answered tokens are distributed as the target's own samples, whatever drafted them. Their log-probabilities under
the target at T are what a GRPO trainer reads as the behaviour logprobs. HIP tensors only; all work is queued on the
current stream of the tensors' device, nothing synchronises with the host.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .embed_op import _FLOATS, _call_on, _ids, _on_gpu
from .head_op import _DT, _p, _workspace


def _seq_rows(x: Tensor, what: str) -> Tensor:
    """x [S, rows, V] with contiguous rows."""
    if x.dtype not in _FLOATS:
        raise NotImplementedError(f"octohead: {what} of dtype {x.dtype} have no HIP kernel")
    return x if x.stride(2) == 1 and x.stride(0) >= 0 and x.stride(1) >= 0 else x.contiguous()


def _verify(logits: Tensor, drafts: Tensor, uniform: Optional[Tensor], draft_logits: Optional[Tensor],
            lengths: Optional[Tensor], inv_T: float, greedy: bool) -> tuple[Tensor, Tensor, Tensor]:
    dev = _on_gpu(logits, drafts, uniform, draft_logits, lengths)
    S, rows, V = logits.shape
    K = rows - 1
    z = _seq_rows(logits, "logits")
    zd = None if draft_logits is None else _seq_rows(draft_logits, "draft logits")
    x = _ids(drafts)
    u = None if uniform is None else uniform.contiguous()
    n = None if lengths is None else _ids(lengths)
    tokens = torch.empty(S, rows, dtype=torch.int64, device=dev)
    accepted = torch.empty(S, dtype=torch.int64, device=dev)
    logp = torch.empty(S, rows, dtype=torch.float32, device=dev)
    nbytes = ctypes.c_size_t(0)
    _lib.call("octo_verify_workspace_bytes", S, K, V, ctypes.byref(nbytes))
    ws = _workspace(nbytes.value, logits)
    _call_on(dev, "octo_verify_drafts", _p(z), z.stride(0), z.stride(1), _p(zd), 0 if zd is None else zd.stride(0),
             0 if zd is None else zd.stride(1), _DT[z.dtype], _p(x), _p(n), _p(u), S, K, V, inv_T, int(greedy),
             _p(tokens), _p(accepted), _p(logp), _p(ws), ws.numel())
    return tokens, accepted, logp


@torch.library.custom_op("octohead::verify_drafts", mutates_args=(), device_types="cuda")
def _verify_op(logits: Tensor, drafts: Tensor, uniform: Optional[Tensor], draft_logits: Optional[Tensor],
               lengths: Optional[Tensor], inv_T: float, greedy: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _verify(logits, drafts, uniform, draft_logits, lengths, inv_T, greedy)


@_verify_op.register_fake
def _(logits, drafts, uniform, draft_logits, lengths, inv_T, greedy):
    S, rows = logits.shape[:2]
    return (logits.new_empty(S, rows, dtype=torch.int64), logits.new_empty(S, dtype=torch.int64),
            logits.new_empty(S, rows, dtype=torch.float32))


def verify_drafts(logits: Tensor, drafts: Tensor, uniform: Optional[Tensor], temperature: float, *,
                  draft_logits: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                  greedy: bool = False) -> tuple[Tensor, Tensor, Tensor]:
    """(tokens [S, K + 1] int64, accepted [S] int64, logp [S, K + 1] fp32): of S sequences the accepted drafts and the
    token drawn behind them, -1 further on; how many were accepted; the target's log-probabilities of the tokens at the
    temperature, 0 further on. K = 0 draws one token a sequence.

    logits [S, K + 1, V] (bf16, f16, fp32): the target's, row i at the position that draft i answers; drafts [S, K];
    uniform [S, K + 1] fp32 in [0, 1): one number a draft and the last for the draw. draft_logits [S, K, V] in the
    logits' type: the distributions that the drafts were sampled from, at the same temperature; None: drafts that were
    not sampled (looked up, or the draft's best). lengths [S]: how many of the K drafts there are (None: all;
    clamped to [0, K]); what lies behind them is not read. greedy:
    a draft is accepted when it is its row's first largest logit, which is also the token behind them; uniform (may be
    None) and draft_logits are not read.

    Decisions and tokens are those of 64-bit probabilities, so the token is the definition's. logp is rounded once from
    64 bits for the drawn token and, below 2^24 logits read, for all; from there on the accepted drafts' and greedy's
    are within 5e-6 before that rounding (their rows' sums are of 32-bit exponentials), and may differ by that between
    calls of other sizes. Nothing is differentiable. A draft outside the vocabulary, or whose draft row has no softmax
    (a NaN, +inf, or every logit masked), is rejected and the token drawn from the target's; where the target's row has
    none, the token is -1 and its logp NaN."""
    if logits.dim() != 3 or not logits.shape[1] or not logits.shape[2]:
        raise ValueError(f"octohead: logits must be [S, K + 1, V], got {tuple(logits.shape)}")
    S, rows, V = logits.shape
    K = rows - 1
    if K > _lib.DRAFTS_MAX:
        raise ValueError(f"octohead: at most {_lib.DRAFTS_MAX} drafts a sequence, got {K}")
    if not temperature > 0 or not 0.0 < 1.0 / float(temperature) < 1e38:
        raise ValueError(f"octohead: temperature {temperature} must be positive and within fp32's range")
    if drafts.shape != (S, K):
        raise ValueError(f"octohead: drafts [{S}, {K}] expected, got {tuple(drafts.shape)}")
    if uniform is None and not greedy:
        raise ValueError("octohead: uniform numbers are needed unless greedy")
    if uniform is not None and (uniform.shape != (S, rows) or uniform.dtype != torch.float32):
        raise ValueError(f"octohead: uniform numbers [{S}, {rows}] in fp32 expected, got {uniform.dtype} "
                         f"{tuple(uniform.shape)}")
    if draft_logits is not None and (draft_logits.shape != (S, K, V) or draft_logits.dtype != logits.dtype):
        raise ValueError(f"octohead: draft logits [{S}, {K}, {V}] in {logits.dtype} expected, got "
                         f"{draft_logits.dtype} {tuple(draft_logits.shape)}")
    if lengths is not None and lengths.shape != (S,):
        raise ValueError(f"octohead: lengths [{S}] expected, got {tuple(lengths.shape)}")
    inv_T = 1.0 / float(temperature)
    if torch.compiler.is_compiling():
        return _verify_op(logits.detach(), drafts, None if uniform is None else uniform.detach(),
                          None if draft_logits is None else draft_logits.detach(), lengths, inv_T, bool(greedy))
    return _verify(logits, drafts, uniform, draft_logits, lengths, inv_T, bool(greedy))
