"""CPU checks of the distillation from a teacher's kept tokens: the fp64 oracle against torch, closed
forms and differences, and the refusals of the Python calls and the C entries."""

import ctypes

import numpy as np
import pytest
import torch

from aspec_amd import _lib, topk_distill_from_logits, topk_distill_fused_grad
from oracle import topk_distill as O


def _case(n=4, vocab=11, k=3, seed=0, temperature=1.0):
    rng = np.random.default_rng(seed)
    x, z = rng.normal(size=(n, vocab)) * 2, rng.normal(size=(n, vocab)) * 2
    logq = torch.log_softmax(torch.as_tensor(z) / temperature, -1).numpy()
    tokens = np.argsort(-z, axis=-1)[:, :k]
    return x, rng.integers(0, vocab, n), tokens, np.take_along_axis(logq, tokens, -1), logq


def test_oracle_against_torch():
    # every token kept: the full divergence, 1 - l1 / 2 and cross-entropy
    x, targets, tokens, logprobs, logq = _case(k=11)
    ce, kl, accept, amax = O.forward(x, targets, tokens, logprobs)
    logp, logq = torch.log_softmax(torch.as_tensor(x), -1), torch.as_tensor(logq)
    np.testing.assert_allclose(kl, torch.nn.functional.kl_div(logp, logq, log_target=True, reduction="none").sum(-1),
                               rtol=1e-12)
    np.testing.assert_allclose(accept, 1 - 0.5 * (logp.exp() - logq.exp()).abs().sum(-1), rtol=1e-12)
    np.testing.assert_allclose(ce, torch.nn.functional.cross_entropy(torch.as_tensor(x), torch.as_tensor(targets),
                                                                     reduction="none"), rtol=1e-12)
    assert amax.tolist() == x.argmax(-1).tolist()
    # the bucket is the divergence of the distributions with the tail as one token
    x, targets, tokens, logprobs, logq = _case(seed=1)
    _, kl, accept, _ = O.forward(x, targets, tokens, logprobs)
    p = np.exp(torch.log_softmax(torch.as_tensor(x), -1).numpy())
    for i in range(len(x)):
        a = np.append(np.exp(logprobs[i]), 1 - np.exp(logprobs[i]).sum())
        b = np.append(p[i, tokens[i]], 1 - p[i, tokens[i]].sum())
        assert abs(kl[i] - (a * np.log(a / b)).sum()) < 1e-12 and abs(accept[i] - np.minimum(a, b).sum()) < 1e-12
    # the same distribution: nothing diverges, everything is accepted
    for tail in ("bucket", "renormalize"):
        _, kl, accept, _ = O.forward(np.where(np.isin(np.arange(11), tokens[0]), logq[0], -np.inf)[None], targets[:1],
                                     tokens[:1], logprobs[:1] - np.log(np.exp(logprobs[0]).sum()), tail)
        assert abs(kl[0]) < 1e-12 and abs(accept[0] - 1) < 1e-12
    # unused slots; a row without any
    tokens = np.array([[2, -1, 5], [-1, -1, -1]])
    _, kl, accept, _ = O.forward(x[:2], targets[:2], tokens, np.log(np.array([[0.5, 9.0, 0.25]] * 2)))
    want = 0.5 * np.log(0.5 / p[0, 2]) + 0.25 * np.log(0.25 / p[0, 5]) + 0.25 * np.log(0.25 / (1 - p[0, 2] - p[0, 5]))
    assert abs(kl[0] - want) < 1e-12 and kl[1] == 0 and accept[1] == 0


@pytest.mark.parametrize("tail", ["bucket", "renormalize"])
@pytest.mark.parametrize("temperature", [1.0, 1.7])
def test_oracle_gradient_against_differences(tail, temperature):
    x, targets, tokens, logprobs, _ = _case(seed=2, temperature=temperature)
    tokens[0, 1], targets[1], targets[2] = -1, -100, tokens[2, 0]
    rng = np.random.default_rng(3)
    g_ce, g_kl = rng.normal(size=4), rng.normal(size=4)

    def loss(x):
        ce, kl, _, _ = O.forward(x, targets, tokens, logprobs, tail, temperature)
        return (g_ce * ce).sum() + (g_kl * kl).sum()

    got, _ = O.grad(x, targets, tokens, logprobs, g_ce, g_kl, tail, temperature)
    step = 1e-6
    for i, j in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i, j] += step
        down[i, j] -= step
        assert abs((loss(up) - loss(down)) / (2 * step) - got[i, j]) < 1e-8


def test_refusals_of_the_calls():
    x, targets = torch.randn(4, 11), torch.tensor([0, 1, 2, 3])
    tokens, logprobs = torch.randint(0, 11, (4, 3)), torch.randn(4, 3) - 5
    ones = torch.ones(4)

    def both(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            topk_distill_from_logits(*args, **kw)
        with pytest.raises(ValueError, match=match):
            topk_distill_fused_grad(*args, ce_weights=ones, kl_weights=ones, **kw)

    both("CUDA logits", x, targets, tokens, logprobs)
    both("tail must be", x, targets, tokens, logprobs, tail="drop")
    for temperature in (0.0, -2.0, float("nan"), float("inf")):
        both("temperature", x, targets, tokens, logprobs, temperature=temperature)
    both("targets must be", x, targets.int(), tokens, logprobs)
    both("targets must be", x, targets[:3], tokens, logprobs)
    both("frozen", x, targets, tokens, logprobs.clone().requires_grad_())
    for t, lp in ((tokens.float(), logprobs), (tokens, logprobs.double()), (tokens, logprobs.bfloat16()),
                  (tokens[:, :2], logprobs), (tokens[:, :0], logprobs[:, :0])):
        both("a teacher is int64 or int32", x, targets, t, lp)
    both("one row per logit row", x, targets, tokens[:3], logprobs[:3])
    rows = torch.tensor([0, 1, 1, 0])
    for r, t, lp in ((rows.int(), tokens, logprobs), (rows[:3], tokens, logprobs),
                     (rows, tokens.view(2, 2, 3), logprobs.view(2, 2, 3)), (rows, tokens[:0], logprobs[:0])):
        both("indexed teacher", x, targets, t, lp, teacher_rows=r)
    with pytest.raises(ValueError, match="go with targets"):
        topk_distill_fused_grad(x, None, tokens, logprobs, ce_weights=ones, kl_weights=ones)
    with pytest.raises(ValueError, match="go with targets"):
        topk_distill_fused_grad(x, targets, tokens, logprobs, kl_weights=ones)
    with pytest.raises(ValueError, match="one value per logit row"):
        topk_distill_fused_grad(x, targets, tokens, logprobs, ce_weights=ones, kl_weights=ones[:2])


def test_refusals_of_the_c_entries():
    lib = _lib.load()
    fake, other = ctypes.c_void_p(4096), ctypes.c_void_p(8192)  # never dereferenced: every call fails its checks

    def calls(dtype=4, rows=2, vocab=100, stride=100, token_dtype=1, kept=5, temperature=1.0, logits=fake, targets=fake,
              tokens=fake, ce=fake, stats=fake, grad=other, grad_stride=100, workspace=None, teacher_rows=None,
              num_teacher_rows=None, which="fwd bwd fused"):
        head = (logits, dtype, rows, vocab, stride, targets, -100, tokens, token_dtype, fake, kept, teacher_rows,
                rows if num_teacher_rows is None else num_teacher_rows)
        if "fwd" in which:
            yield lib.aspec_topk_distill_fwd(*head, 0, temperature, ce, fake, fake, None, stats, workspace, None, None)
        if "bwd" in which:
            yield lib.aspec_topk_distill_bwd(*head, temperature, stats, fake, fake, grad, grad_stride, None)
        if "fused" in which:
            yield lib.aspec_topk_distill_fused_fwd_bwd(*head, 0, temperature, fake, fake, ce, fake, fake, None, stats,
                                                       workspace, grad, grad_stride, None, None)

    def refused(error, match, **kw):
        for status in calls(**kw):
            with pytest.raises(error, match=match):
                _lib.check(status)

    refused(NotImplementedError, "bf16, fp16 or fp32", dtype=1)
    for bad in ({"rows": -1}, {"vocab": 0}, {"stride": 99}):
        refused(ValueError, "at least as far apart", **bad)
    refused(ValueError, "at least as far apart", grad_stride=99, which="bwd fused")
    refused(NotImplementedError, "524288", vocab=524289, stride=524289)
    refused(ValueError, "int64 or int32", token_dtype=4)
    refused(ValueError, "a teacher token per row", kept=0)
    refused(NotImplementedError, "128", kept=129)
    refused(ValueError, "a table of at least one", teacher_rows=fake, num_teacher_rows=0)
    refused(ValueError, "a table of at least one", num_teacher_rows=3)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-45, 3e38):
        refused(ValueError, "temperature", temperature=temperature)
    for bad in ({"logits": None}, {"tokens": None}):
        refused(ValueError, "null pointer", **bad)
    refused(ValueError, "null pointer", stats=None, which="bwd")
    refused(ValueError, "null pointer", ce=None, which="fwd fused")
    refused(ValueError, "null pointer", grad=None, which="bwd fused")
    refused(ValueError, "null pointer", targets=None, which="bwd fused")  # a gradient of ce without a target
    refused(ValueError, "null pointer", vocab=151936, stride=151936, rows=1, which="fwd")  # parts without a workspace
    refused(ValueError, "in place", grad=fake, grad_stride=101, which="bwd fused")
    assert all(status == 0 for status in calls(rows=0))
    size = ctypes.c_size_t(1)
    assert lib.aspec_topk_distill_workspace_bytes(4, 8192, 32000, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.aspec_topk_distill_workspace_bytes(4, 16, 32000, ctypes.byref(size)) == 0 and size.value > 0


def test_refusals_of_the_check_entry():
    lib = _lib.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks, or has no rows

    def check(rows=2, vocab=100, tokens=fake, token_dtype=1, logprobs=fake, kept=5, teacher_rows=None,
              num_teacher_rows=None, words=fake):
        _lib.check(lib.aspec_topk_distill_check(
            rows, vocab, fake, -100, tokens, token_dtype, logprobs, kept, teacher_rows,
            rows if num_teacher_rows is None else num_teacher_rows, words, None))

    for error, match, bad in (
            (ValueError, "at least as far apart", {"rows": -1}), (ValueError, "at least as far apart", {"vocab": 0}),
            (NotImplementedError, "524288", {"vocab": 524289}), (ValueError, "int64 or int32", {"token_dtype": 4}),
            (ValueError, "a teacher token per row", {"kept": 0}), (NotImplementedError, "128", {"kept": 129}),
            (ValueError, "a table of at least one", {"teacher_rows": fake, "num_teacher_rows": 0}),
            (ValueError, "a table of at least one", {"num_teacher_rows": 3}),
            (ValueError, "null pointer", {"tokens": None}), (ValueError, "null pointer", {"logprobs": None}),
            (ValueError, "null pointer", {"words": None})):
        with pytest.raises(error, match=match):
            check(**bad)
    check(rows=0)
