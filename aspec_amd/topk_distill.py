"""Distillation from a teacher of which only the best tokens were kept, on the HIP kernels of
csrc/topk_distill.hip and csrc/topk_distill_fused.hip.

The full-vocabulary losses (`aspec_amd.loss`, the reference's `_prediction_terms`,
aspec/models/dspark.py:553-612) need the teacher's logits [rows, V]. A cache keeps K pairs (token,
log-probability) of a teacher row instead, as `aspec_amd.token_logprobs.token_logprobs(top_k=K)`
writes them, and the divergence is taken over those tokens:

  p = softmax(logits / temperature), q = the teacher's kept probabilities, r = its mass outside them,
  R = the student's mass outside them
  tail="bucket":       kl = sum q (log q - log p) + r (log r - log R): the tokens outside as one event
                       (a lower bound of the full divergence, exact as r goes to 0)
  tail="renormalize":  kl = sum q' (log q' - log p), q' = q / sum q
  accept_rate = sum min(p, q) + min(r, R): the probability that a token drafted from p is accepted
                by the teacher (1 - l1 / 2 of the full losses; an upper bound in the bucket)
  ce = cross-entropy of the hard target at temperature 1

No reference function matches. No CPU path: the HIP library runs or the call raises.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from aspec_amd import _lib
from aspec_amd._launch import check_first, index_flags, launch, settle
from aspec_amd.token_logprobs import LOGIT_CODES, check_temperature, float_grad, logit_rows, row_stride, vector

_TAILS = {"bucket": 0, "renormalize": 1}
_TOKEN_CODES = {torch.int64: 1, torch.int32: 2}  # ASPEC_MASK_* codes of the teacher's tokens


class _Call:
    """The checked arguments of one call: what the forward, the gradient and the one-pass entry share."""

    def __init__(self, logits, targets, teacher_indices, teacher_logprobs, teacher_rows, tail, temperature,
                 ignore_index):
        self.temperature = check_temperature(temperature)
        if tail not in _TAILS:
            raise ValueError(f"tail must be 'bucket' or 'renormalize', got {tail!r}")
        self.renormalize = _TAILS[tail]
        self.ignore_index = int(ignore_index)
        lead, dev = logits.shape[:-1], logits.device
        rows = logits.numel() // max(logits.shape[-1] if logits.ndim else 0, 1)
        if targets is not None:
            if targets.dtype != torch.int64 or targets.numel() != rows or targets.device != dev:
                raise ValueError("targets must be one int64 class index per logit row on the logits device")
            targets = vector(targets)
        if teacher_logprobs.requires_grad:
            raise ValueError("top-logit distillation requires a frozen teacher")
        if (teacher_indices.dtype not in _TOKEN_CODES or teacher_logprobs.dtype != torch.float32
                or teacher_indices.ndim < 1 or teacher_indices.shape != teacher_logprobs.shape
                or teacher_indices.shape[-1] == 0
                or teacher_indices.device != dev or teacher_logprobs.device != dev):
            raise ValueError("a teacher is int64 or int32 tokens and FP32 log-probabilities of one shape "
                             "[..., K >= 1] on the logits device")
        kept = teacher_indices.shape[-1]
        if teacher_rows is not None:
            if (teacher_indices.ndim != 2 or (teacher_indices.shape[0] == 0 and rows)
                    or teacher_rows.dtype != torch.int64 or teacher_rows.numel() != rows or teacher_rows.device != dev):
                raise ValueError("indexed teacher requires a nonempty 2D table and one int64 index per row "
                                 "on the logits device")
            teacher_rows = vector(teacher_rows)
        elif teacher_indices.shape[:-1] != lead and teacher_indices.shape[:-1] != (rows,):
            raise ValueError("a teacher without teacher_rows has one row per logit row")
        self.lead, self.rows = lead, rows
        self.targets, self.teacher_rows = targets, teacher_rows
        self.indices, self.logprobs = (t if t.ndim == 2 and t.is_contiguous() else t.reshape(-1, kept).contiguous()
                                       for t in (teacher_indices, teacher_logprobs))

    def tensors(self):
        return self.targets, self.indices, self.logprobs, self.teacher_rows

    def head(self, flat):
        return _head(flat, self.targets, self.ignore_index, self.indices, self.logprobs, self.teacher_rows)

    def check(self, flat, flags, waits):
        """The flags that are left to the logits' pass. Where the call `waits` for its check, the indices of
        a long pass are checked ahead of it."""
        if not waits or not check_first(flags, flat):
            return flags
        launch("topk_distill_check", flat.device, flags, "aspec_topk_distill_check", *flat.shape,
               _lib.ptr(self.targets), self.ignore_index, self.indices.data_ptr(), _TOKEN_CODES[self.indices.dtype],
               self.logprobs.data_ptr(), self.indices.shape[1], _lib.ptr(self.teacher_rows), self.indices.shape[0],
               flags.ptr)
        return None

    def outputs(self, flat, want_argmax, want_stats):
        """(ce, kl, accept_rate, argmax, stats, workspace) to be written; None where not wanted."""
        dev, lead = flat.device, self.lead
        work_bytes, stat_floats = _sizes(LOGIT_CODES[flat.dtype], *flat.shape)
        return (torch.empty(lead, dtype=torch.float32, device=dev) if self.targets is not None else None,
                torch.empty(lead, dtype=torch.float32, device=dev), torch.empty(lead, dtype=torch.float32, device=dev),
                torch.empty(lead, dtype=torch.int64, device=dev) if want_argmax else None,
                torch.empty((self.rows, stat_floats), dtype=torch.float32, device=dev) if want_stats else None,
                torch.empty(work_bytes, dtype=torch.uint8, device=dev) if work_bytes else None)


@functools.lru_cache(maxsize=256)
def _sizes(dtype: int, rows: int, vocab: int) -> tuple[int, int]:
    """(workspace bytes, floats of statistics per row) of a call."""
    lib, size = _lib.load(), ctypes.c_size_t()
    _lib.check(lib.aspec_topk_distill_workspace_bytes(dtype, rows, vocab, ctypes.byref(size)))
    return size.value, lib.aspec_topk_distill_stats_floats()


def _head(flat, targets, ignore_index, indices, logprobs, teacher_rows):
    """The arguments that every entry begins with."""
    return (flat.data_ptr(), LOGIT_CODES[flat.dtype], flat.shape[0], flat.shape[1], row_stride(flat), _lib.ptr(targets),
            ignore_index, indices.data_ptr(), _TOKEN_CODES[indices.dtype], logprobs.data_ptr(), indices.shape[1],
            _lib.ptr(teacher_rows), indices.shape[0])


def _read_twice(flat) -> bool:
    """Whether the one-pass entry makes two passes over such rows, with statistics between them."""
    return _lib.load().aspec_topk_distill_reads(LOGIT_CODES[flat.dtype], flat.shape[1]) > 1


def _forward(logits, call, want_argmax, check, has_backward):
    """One forward launch: (results, logit rows, statistics, index flags to be settled)."""
    flat = logit_rows(logits, "top-logit distillation")
    ce, kl, accept, amax, stats, workspace = call.outputs(flat, want_argmax, has_backward)
    flags = index_flags(check, flat.device)
    pass_flags, ptr = call.check(flat, flags, not has_backward), _lib.ptr
    launch("topk_distill_fwd", flat.device, pass_flags, "aspec_topk_distill_fwd", *call.head(flat), call.renormalize,
           call.temperature, ptr(ce), kl.data_ptr(), accept.data_ptr(), ptr(amax), ptr(stats), ptr(workspace),
           None if pass_flags is None else pass_flags.ptr)
    return (ce, kl, accept, amax), flat, stats, flags


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call, want_argmax, check):
        out, flat, stats, ctx.flags = _forward(logits, call, want_argmax, check, True)
        ctx.save_for_backward(flat, stats, *call.tensors())
        ctx.parameters = (call.ignore_index, call.temperature, logits.shape)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in out[2:] if t is not None))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_ce, g_kl, *_):
        flat, stats, targets, indices, logprobs, teacher_rows = ctx.saved_tensors
        ignore_index, temperature, shape = ctx.parameters
        g_ce, g_kl = float_grad(g_ce), float_grad(g_kl)
        grad = torch.empty(flat.shape, dtype=flat.dtype, device=flat.device)
        launch("topk_distill_bwd", flat.device, None, "aspec_topk_distill_bwd",
               *_head(flat, targets, ignore_index, indices, logprobs, teacher_rows), temperature, stats.data_ptr(), _lib.ptr(g_ce), _lib.ptr(g_kl), grad.data_ptr(), flat.shape[1])
        # the forward's flags, read with this backward's kernel already queued
        settle(ctx.flags)
        return grad if grad.shape == shape else grad.view(shape), None, None, None


def topk_distill_from_logits(logits, targets, teacher_indices, teacher_logprobs, *, teacher_rows=None, tail="bucket",
                             temperature=1.0, ignore_index=-100, return_argmax=False, check_indices=True):
    """Per-row fp32 (ce, kl, accept_rate[, argmax]) of logits [..., V] (bf16, fp16 or fp32, V <= 524288)
    in one read; `ce` and `kl` are differentiable in `logits` (one read and one write).

    `targets` [...] int64 (`ignore_index`: ce 0, no gradient) or None (ce is None).
    `teacher_indices` (int64 or int32) and `teacher_logprobs` (fp32) [..., K], K <= 128, hold a frozen
    teacher's kept tokens and their log-probabilities at `temperature`, in any order, each token once;
    index -1 is an unused slot. With `teacher_rows` [...] int64 they are a [T, K] table addressed per
    row. A row without any token has kl 0, accept_rate 0 and no gradient of kl. In the bucket a
    remaining mass up to 2^-20 counts as the rounding of the log-probabilities, that is as none.

    Logits of -inf are tokens without probability: a kept one, or a whole tail that the teacher gives
    mass, makes kl infinite, as the definition has it, with finite gradients. A row of nothing else
    has infinite losses and a zero gradient; one with a NaN or +inf has NaN.

    A target, teacher token or teacher row out of range, or a token twice in a row, gives a NaN row
    (losses and gradient; a bad target: ce and gradient) and raises ValueError: before the call
    returns, or, where `logits` requires grad, from the backward, behind its kernel. Reading that
    check waits for the GPU: with `check_indices=False` nothing waits, and the NaN is the only sign.
    So it is in a call that is captured into a graph."""
    call = _Call(logits, targets, teacher_indices, teacher_logprobs, teacher_rows, tail, temperature, ignore_index)
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TopkDistill.apply(logits, call, return_argmax, check_indices)
    else:
        out, _, _, flags = _forward(logits, call, return_argmax, check_indices, False)
        settle(flags)
    return out if return_argmax else out[:3]


def topk_distill_fused_grad(logits, targets, teacher_indices, teacher_logprobs, *, ce_weights=None, kl_weights,
                            teacher_rows=None, tail="bucket", temperature=1.0, ignore_index=-100, return_argmax=False,
                            in_place=False, check_indices=True):
    """`topk_distill_from_logits` and dlogits of sum_r (ce_weights[r] ce[r] + kl_weights[r] kl[r]) from
    one read of the logits (no autograd): (ce, kl, accept_rate, dlogits[, argmax]). `ce_weights` goes
    with `targets`. With `in_place` the dlogits overwrite `logits`, which then are rows of adjacent
    elements. Rows too long for one workgroup (V > 163840, fp32: 81920) are read twice."""
    out, flags = _fused(logits, targets, teacher_indices, teacher_logprobs, ce_weights, kl_weights, teacher_rows, tail,
                        temperature, ignore_index, return_argmax, in_place, check_indices, True)
    settle(flags)
    return out if return_argmax else out[:4]


def _fused(logits, targets, teacher_indices, teacher_logprobs, ce_weights, kl_weights, teacher_rows, tail, temperature,
           ignore_index, return_argmax, in_place, check_indices, waits):
    """The launch behind `topk_distill_fused_grad`, its index flags still to be settled: at once (`waits`),
    or behind work that the caller queues first."""
    call = _Call(logits, targets, teacher_indices, teacher_logprobs, teacher_rows, tail, temperature, ignore_index)
    if (targets is None) != (ce_weights is None):
        raise ValueError("ce_weights go with targets")
    weights = []
    for w in (ce_weights, kl_weights):
        if w is not None and (w.numel() != call.rows or w.device != logits.device):
            raise ValueError("objective weights must hold one value per logit row on the logits device")
        weights.append(None if w is None else vector(w.detach()).to(torch.float32))
    logits = logits.detach()
    flat = logit_rows(logits, "top-logit distillation")
    if in_place and flat.data_ptr() != logits.data_ptr():
        raise ValueError("in_place needs logits whose rows are evenly spaced and their elements adjacent")
    ce, kl, accept, amax, stats, workspace = call.outputs(flat, return_argmax, _read_twice(flat))
    grad = flat if in_place else torch.empty(flat.shape, dtype=flat.dtype, device=flat.device)
    flags = index_flags(check_indices, flat.device)
    pass_flags, ptr = call.check(flat, flags, waits), _lib.ptr
    launch("topk_distill_fused", flat.device, pass_flags, "aspec_topk_distill_fused_fwd_bwd", *call.head(flat),
           call.renormalize, call.temperature, ptr(weights[0]), ptr(weights[1]), ptr(ce), kl.data_ptr(),
           accept.data_ptr(), ptr(amax), ptr(stats), ptr(workspace), grad.data_ptr(), row_stride(grad),
           None if pass_flags is None else pass_flags.ptr)
    if in_place and not logits.is_inference():
        torch.autograd.graph.increment_version(logits)  # a graph that kept the logits must not use them
    return (ce, kl, accept, logits if in_place else grad.view(logits.shape), amax), flags
