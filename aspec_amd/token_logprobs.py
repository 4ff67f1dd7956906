"""Log-probabilities of given tokens, entropy and the best alternatives of rows of logits, on the
HIP kernels of csrc/token_logprobs.hip.

What a scoring or verifying model answers with, and what a distillation cache keeps of a teacher
(`aspec_amd.topk_distill` trains against `top_indices` / `top_logprobs`). One read of the logits
forward, one read and one write backward:

  logp          = log_softmax(logits / temperature)
  logprobs      = logp[token]
  entropy       = -sum p logp
  top_logprobs  = the top_k largest logp, descending; ties by the lower token index

No reference function matches: the reference's target engine returns hidden states, and its head
takes the teacher's logits whole (aspec/models/dspark.py:553-612). No CPU path: the HIP library runs
or the call raises.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from aspec_amd import _lib
from aspec_amd._launch import check_first, index_flags, launch, settle

# ASPEC_MASK_* codes of the logits' types
LOGIT_CODES = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}


class TokenLogprobs(NamedTuple):
    """Per row: fp32 `logprobs` (None without token ids), fp32 `entropy`, and, with top_k > 0, fp32
    `top_logprobs` and int64 `top_indices` [..., top_k] (else None)."""

    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def logit_rows(logits: torch.Tensor, what: str) -> torch.Tensor:
    """[rows, V] of logits [..., V]: a view where the rows are evenly spaced and their elements
    adjacent (rows padded to a longer stride among them), else a contiguous copy."""
    if not logits.is_cuda:
        raise ValueError(f"{what} requires CUDA logits")
    if logits.dtype not in LOGIT_CODES:
        raise ValueError(f"{what} requires BF16, FP16 or FP32 logits")
    if logits.ndim < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what} requires logits with a vocabulary dimension")
    vocab = logits.shape[-1]
    rows = logits.numel() // vocab
    flat = logits if logits.ndim == 2 else logits.reshape(rows, vocab)
    if rows and (flat.stride(-1) != 1 and vocab > 1 or flat.stride(0) < vocab and rows > 1):
        flat = flat.contiguous()  # transposed or broadcast rows
    return flat


def row_stride(flat: torch.Tensor) -> int:
    return flat.stride(0) if flat.shape[0] > 1 else flat.shape[1]


def vector(t: torch.Tensor) -> torch.Tensor:
    """A per-row argument as one contiguous vector."""
    return t if t.ndim == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def float_grad(g: torch.Tensor | None) -> torch.Tensor | None:
    """An upstream gradient as the kernels read it."""
    if g is None or (g.dtype == torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


def check_temperature(temperature) -> float:
    temperature = float(temperature)
    if not (math.isfinite(temperature) and temperature > 0.0):
        raise ValueError(f"temperature must be finite and > 0, got {temperature}")
    return temperature


@functools.lru_cache(maxsize=256)
def _sizes(dtype: int, rows: int, vocab: int, top_k: int) -> tuple[int, int]:
    """(workspace bytes, floats of statistics per row) of a call."""
    lib, size = _lib.load(), ctypes.c_size_t()
    _lib.check(lib.aspec_token_logprobs_workspace_bytes(dtype, rows, vocab, top_k, ctypes.byref(size)))
    return size.value, lib.aspec_token_logprobs_stats_floats()


def _head(flat, ids, ignore_index, temperature, top_k):
    """The arguments that both entries begin with."""
    return (flat.data_ptr(), LOGIT_CODES[flat.dtype], flat.shape[0], flat.shape[1], row_stride(flat), _lib.ptr(ids),
            ignore_index, temperature, top_k)


def _forward(logits, ids, top_k, temperature, ignore_index, check_ids, has_backward):
    """One forward launch: (results, logit rows, statistics, index flags to be settled)."""
    flat = logit_rows(logits, "token_logprobs")
    rows, vocab = flat.shape
    dev, lead = flat.device, logits.shape[:-1]
    work_bytes, stat_floats = _sizes(LOGIT_CODES[flat.dtype], rows, vocab, top_k)
    workspace = torch.empty(work_bytes, dtype=torch.uint8, device=dev) if work_bytes else None
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    logprobs = torch.empty(lead, dtype=torch.float32, device=dev) if ids is not None else None
    top = torch.empty((*lead, top_k), dtype=torch.float32, device=dev) if top_k else None
    top_indices = torch.empty((*lead, top_k), dtype=torch.int64, device=dev) if top_k else None
    stats = torch.empty((rows, stat_floats), dtype=torch.float32, device=dev) if has_backward else None
    flags = index_flags(check_ids and ids is not None, dev)
    pass_flags, ptr = flags, _lib.ptr
    if not has_backward and check_first(flags, flat):
        launch("token_logprobs_check", dev, flags, "aspec_token_logprobs_check", ids.data_ptr(), rows, vocab,
               ignore_index, flags.ptr)
        pass_flags = None
    launch("token_logprobs_fwd", dev, pass_flags, "aspec_token_logprobs_fwd",
           *_head(flat, ids, ignore_index, temperature, top_k), ptr(logprobs), entropy.data_ptr(), ptr(top),
           ptr(top_indices), ptr(stats), ptr(workspace), None if pass_flags is None else pass_flags.ptr)
    return (logprobs, entropy, top, top_indices), flat, stats, flags


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, top_k, temperature, ignore_index, check_ids):
        out, flat, stats, ctx.flags = _forward(logits, ids, top_k, temperature, ignore_index, check_ids, True)
        ctx.save_for_backward(flat, ids, out[3], stats)
        ctx.parameters = (ignore_index, temperature, top_k)
        ctx.shape = logits.shape
        ctx.set_materialize_grads(False)
        if out[3] is not None:
            ctx.mark_non_differentiable(out[3])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_top, _):
        flat, ids, top_indices, stats = ctx.saved_tensors
        g_logprobs, g_entropy, g_top = map(float_grad, (g_logprobs, g_entropy, g_top))
        grad = torch.empty(flat.shape, dtype=flat.dtype, device=flat.device)
        ptr = _lib.ptr
        launch("token_logprobs_bwd", flat.device, None, "aspec_token_logprobs_bwd",
               *_head(flat, ids, *ctx.parameters), ptr(top_indices), stats.data_ptr(), ptr(g_logprobs), ptr(g_entropy), ptr(g_top), grad.data_ptr(), flat.shape[1])
        # the forward's flags, read with this backward's kernel already queued
        settle(ctx.flags)
        return grad if grad.shape == ctx.shape else grad.view(ctx.shape), None, None, None, None, None


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor | None = None, *, top_k: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100, check_ids: bool = True) -> TokenLogprobs:
    """`TokenLogprobs` of logits [..., V] (bf16, fp16 or fp32, V <= 524288) in fp32, differentiable in
    `logits` through `logprobs`, `entropy` and `top_logprobs`.

    `token_ids` [...] int64: one token per row; `ignore_index` gives logprob 0 without a gradient. A
    token outside [0, V) gives a NaN logprob (and a NaN gradient row) and raises ValueError: before
    the call returns, or, where `logits` requires grad, from the backward, behind its kernel. Reading
    that check waits for the GPU: with `check_ids=False` nothing waits, and the NaN is the only sign.
    So it is in a call that is captured into a graph.

    `top_k` (at most 128 and V) alternatives per row, by logit, ties by the lower index, NaN first.
    Logits of -inf are tokens without probability (logprob -inf). A row of nothing else has logprob
    -inf, entropy 0 and a zero gradient; one with a NaN or +inf has NaN results."""
    temperature = check_temperature(temperature)
    if isinstance(top_k, bool) or int(top_k) != top_k or top_k < 0:
        raise ValueError(f"top_k must be a whole number >= 0, got {top_k}")
    rows = logits.numel() // max(logits.shape[-1] if logits.ndim else 0, 1)
    if token_ids is not None:
        if token_ids.dtype != torch.int64 or token_ids.device != logits.device or (
                token_ids.shape != logits.shape[:-1] and token_ids.shape != (rows,)):
            raise ValueError("token_ids must be one int64 token per logit row on the logits device")
        token_ids = vector(token_ids)
    args = (logits, token_ids, int(top_k), temperature, int(ignore_index), check_ids)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(*args))
    out, _, _, flags = _forward(*args, False)
    settle(flags)
    return TokenLogprobs(*out)
