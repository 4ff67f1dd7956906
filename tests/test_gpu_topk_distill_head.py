"""Where the distillation from a teacher's kept tokens is used: the head's objective
(`selective_head_distillation`) and the DSpark head terms (`dspark_prediction_terms` with
`cached_target_topk`), and the run from a teacher's pass through its cache to a training step.

The head's GEMMs are the library's on bf16 operands. The losses are held to the fp64 oracle on the
logits as the GEMM rounded them; dh to the product, in fp64, of the bf16 gradient of those logits,
whose rounding is half a step (2^-8) per element, with W, and rounded once more."""

import numpy as np
import pytest
import torch

from aspec_amd import (acceptance_statistics, dspark_prediction_terms, selective_head_distillation, token_logprobs,
                       topk_distill_from_logits)
from oracle import topk_distill as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEPS = U * (128 + 4 * 60)  # a probability's relative error, as in test_gpu_topk_distill.py


def _case(gpu, rows, hidden, vocab, top, dtype=torch.bfloat16, seed=0, trows=0):
    g = torch.Generator(device=gpu).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=gpu, generator=g) * scale).to(dtype)

    w = normal(vocab, hidden, scale=0.2)
    teacher = normal(trows or rows, hidden)
    index = torch.randint(0, trows, (rows,), device=gpu, generator=g) if trows else None
    h = ((teacher[index] if trows else teacher).float() + 0.5 * torch.randn(rows, hidden, device=gpu, generator=g)).to(dtype)
    cache = token_logprobs(teacher @ w.t(), top_k=top)  # the teacher's pass
    targets = torch.randint(0, vocab, (rows,), device=gpu, generator=g)
    targets[::5] = -100
    ce_w, kl_w = (torch.rand(rows, device=gpu, generator=g) for _ in range(2))
    kl_w[3::7] = 0
    return h, w, targets, cache.top_indices, cache.top_logprobs, index, ce_w, kl_w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab,trows", [(1000, 0), (5003, 12), (33000, 0)])
def test_objective(gpu, dtype, vocab, trows):
    h, w, targets, tokens, logprobs, index, ce_w, kl_w = _case(gpu, 40, 256, vocab, 24, dtype, vocab, trows)
    leaf = h.clone().requires_grad_()
    objective, ce, kl, accept, amax = selective_head_distillation(
        leaf, w, targets, tokens, logprobs, ce_weights=ce_w, kl_weights=kl_w, teacher_rows=index, return_argmax=True)
    (3.0 * objective).backward()
    logits = h @ w.t()
    at = index.cpu().numpy() if index is not None else slice(None)
    args = (logits.double().cpu().numpy(), targets.cpu().numpy(), tokens.cpu().numpy()[at],
            logprobs.double().cpu().numpy()[at])
    r_ce, r_kl, r_accept, r_amax = O.forward(*args)
    np.testing.assert_allclose(ce.double().cpu(), r_ce, atol=2 * STEPS, rtol=8 * U)
    np.testing.assert_allclose(kl.double().cpu(), r_kl, atol=3 * STEPS, rtol=3 * STEPS)
    np.testing.assert_allclose(accept.double().cpu(), r_accept, atol=2 * STEPS)
    assert np.array_equal(amax.cpu().numpy(), r_amax)
    want = (ce_w.double().cpu().numpy() * r_ce).sum() + (kl_w.double().cpu().numpy() * r_kl).sum()
    # two dot products of 40 terms
    assert abs(objective.item() - want) <= (4 * STEPS + 80 * U) * (1 + abs(want)) * 2
    dlogits, size = O.grad(*args, ce_w.double().cpu().numpy(), kl_w.double().cpu().numpy())
    w64 = w.double().cpu().numpy()
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    tiny = 0.0 if dtype == torch.bfloat16 else 2.0 ** -25  # half a step below fp16's normal range
    dh, bound = dlogits @ w64, (half * np.abs(dlogits) + 3 * STEPS * size + tiny) @ np.abs(w64)
    bound += vocab * U * (np.abs(dlogits) @ np.abs(w64))  # the GEMM's fp32 sums
    got = leaf.grad.double().cpu().numpy()
    # two roundings of dh: the GEMM's and the scale's
    assert (np.abs(got - 3.0 * dh) <= 3.0 * bound * (1 + 2 * half) + 2 * half * np.abs(3.0 * dh) + tiny).all()
    assert not (ce.requires_grad or kl.requires_grad or accept.requires_grad)


def test_objective_without_targets_and_refusals(gpu):
    h, w, targets, tokens, logprobs, index, ce_w, kl_w = _case(gpu, 16, 128, 2000, 8)
    leaf = h.clone().requires_grad_()
    both = selective_head_distillation(leaf, w, targets, tokens, logprobs, ce_weights=0 * ce_w, kl_weights=kl_w)
    alone = selective_head_distillation(leaf, w, None, tokens, logprobs, kl_weights=kl_w)
    assert alone[1] is None and torch.equal(alone[2], both[2])
    (a,), (b,) = (torch.autograd.grad(o[0], leaf) for o in (both, alone))
    assert torch.equal(a, b)
    bad = tokens.clone()
    bad[3, 2] = 2000
    with torch.no_grad(), pytest.raises(ValueError, match="teacher token out of range"):
        selective_head_distillation(leaf, w, None, bad, logprobs, kl_weights=kl_w)
    out = selective_head_distillation(leaf, w, None, bad, logprobs, kl_weights=kl_w)
    with pytest.raises(ValueError, match="teacher token out of range"):
        out[0].backward()
    with pytest.raises(ValueError, match="share H"):
        selective_head_distillation(h[:, :64], w, None, tokens, logprobs, kl_weights=kl_w)
    with pytest.raises(ValueError, match="frozen"):
        selective_head_distillation(h, w.clone().requires_grad_(), None, tokens, logprobs, kl_weights=kl_w)
    with pytest.raises(ValueError, match="go with targets"):
        selective_head_distillation(h, w, targets, tokens, logprobs, kl_weights=kl_w)


@pytest.mark.parametrize("table", [False, True])
def test_prediction_terms(gpu, table):
    """The head terms from a cached teacher: the pass's own losses, weighted and counted as with a full
    teacher."""
    batch, blocks, width, context, top, vocab = 2, 3, 4, 10, 12, 3000
    g = torch.Generator(device=gpu).manual_seed(5)
    w = (torch.randn(vocab, 64, device=gpu, generator=g) * 0.2).to(torch.bfloat16)
    states = torch.randn(batch, context, 64, device=gpu, generator=g).to(torch.bfloat16)
    cache = token_logprobs(states @ w.t(), top_k=top)
    positions = torch.randint(0, context, (batch, blocks, width), device=gpu, generator=g)
    rows = torch.arange(batch, device=gpu)[:, None, None]
    hidden = (states[rows, positions].float() + 0.3 * torch.randn(batch, blocks, width, 64, device=gpu, generator=g)
              ).to(torch.bfloat16)
    targets = cache.top_indices[rows, positions, 0]
    targets[0, 0] = torch.randint(0, vocab, (width,), device=gpu, generator=g)
    mask = (torch.rand(batch, blocks, width, device=gpu, generator=g) > 0.2).float()
    weights = mask * torch.rand(batch, blocks, width, device=gpu, generator=g)
    topk = (cache.top_indices, cache.top_logprobs)
    if not table:
        topk = tuple(t[rows, positions] for t in topk)
    leaf = hidden.clone().requires_grad_()
    terms = dspark_prediction_terms(leaf, targets, targets, w, None, mask, weights, cached_target_topk=topk,
                                    cached_target_positions=positions if table else None)
    ce_num, kl_num, conf, position_loss, position_correct, totals = terms
    logits = (hidden.reshape(-1, 64) @ w.t()).requires_grad_()
    per_row = [t[rows, positions].reshape(-1, top) for t in (cache.top_indices, cache.top_logprobs)]
    ce, kl, accept, amax = topk_distill_from_logits(logits, targets.reshape(-1), *per_row, return_argmax=True)
    assert ce_num.item() == (ce.view_as(weights) * weights).sum().item()
    assert kl_num.item() == (kl.view_as(weights) * weights).sum().item() and conf.item() == 0
    assert torch.equal(position_loss, (ce.detach().view_as(mask) * mask).sum((0, 1)))
    assert torch.equal(position_correct, ((amax.view_as(targets) == targets) & (mask > 0.5)).float().sum((0, 1)))
    assert torch.equal(totals, acceptance_statistics(accept.view_as(mask), mask))
    (dh,) = torch.autograd.grad(ce_num + 0.5 * kl_num, leaf)
    v = weights.reshape(-1)
    (dx,) = torch.autograd.grad([ce, kl], logits, [v, 0.5 * v])
    torch.testing.assert_close(dh.reshape(-1, 64), dx @ w, atol=1e-5, rtol=2.0 ** -7)
    with pytest.raises(ValueError, match="cached_target_topk is the teacher"):
        dspark_prediction_terms(leaf, targets, targets, w, hidden, mask, weights, cached_target_topk=topk)
    if table:
        with pytest.raises(ValueError, match="teacher table"):
            dspark_prediction_terms(leaf, targets, targets, w, None, mask, weights, cached_target_positions=positions,
                                    cached_target_topk=tuple(t[0] for t in topk))


def test_training_step_from_a_cache(gpu):
    """A teacher's pass, its cache moved through int32 on the host as a file would hold it, and training
    steps of the head's hidden states captured into one graph: replays equal the eager step."""
    h, w, targets, tokens, logprobs, index, ce_w, kl_w = _case(gpu, 32, 128, 4000, 16, seed=9, trows=20)
    stored = tokens.int().cpu(), logprobs.cpu()
    tokens, logprobs = (t.to(gpu) for t in stored)
    wt = w.t().contiguous()

    def step(x):
        leaf = x.detach().requires_grad_()
        out = selective_head_distillation(leaf, w, targets, tokens, logprobs, ce_weights=ce_w, kl_weights=kl_w,
                                          teacher_rows=index, weight_t=wt)
        (dh,) = torch.autograd.grad(out[0], leaf)
        return [t.detach() for t in (*out, dh)]

    static = h.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(static)
    for i in range(3):
        fresh = _case(gpu, 32, 128, 4000, 16, seed=20 + i, trows=20)[0]
        static.copy_(fresh)
        graph.replay()
        want = step(fresh)
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
