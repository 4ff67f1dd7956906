"""Distillation from a teacher's kept tokens on the GPU against the fp64 oracle: losses, acceptance,
argmax and the gradient, through autograd and in one pass.

Tolerances (u = 2^-24, half a step of fp32): a row sum is at most 96 rounded additions deep and an
exponent of size d <= 60 that weighs anything carries 4 u d and v_exp_f32 a step, so a probability, or
the ratio of two sums, is off by at most STEPS = u (128 + 4 * 60) relative. kl takes two such sums and
is formed in 64 bits from there; its terms and the gradient's are weighted by probabilities, and the
gradient is rounded once to its type."""

import numpy as np
import pytest
import torch

from aspec_amd import token_logprobs, topk_distill_from_logits, topk_distill_fused_grad
from oracle import topk_distill as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEPS = U * (128 + 4 * 60)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}  # below the normal range
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _close(got, ref, tol, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == ref.shape, what
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - ref) <= tol))
    assert not bad.any(), (what, np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5])


class Case:
    """Student rows near teacher rows; the teacher's `kept` best tokens, in shuffled order."""

    def __init__(self, gpu, rows, vocab, kept, dtype, seed, *, table=0, temperature=1.0, fewer=True):
        g = torch.Generator(device=gpu).manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, device=gpu, generator=g)

        trows = table or rows
        z = normal(trows, vocab) * 2
        z[:, : min(vocab, 3)] += 8 * torch.rand(trows, min(vocab, 3), device=gpu, generator=g)
        self.rows = torch.randint(0, trows, (rows,), device=gpu, generator=g) if table else None
        top = torch.log_softmax(z.double() / temperature, -1).topk(kept, dim=-1)
        order = torch.rand(trows, kept, device=gpu, generator=g).argsort(-1)
        self.logprobs, self.tokens = top.values.float().gather(1, order), top.indices.gather(1, order)
        if fewer and kept > 2:
            self.tokens[0, 1:3] = -1
            self.tokens[-1] = -1
        self.x = ((z[self.rows] if table else z) + normal(rows, vocab)).to(dtype)
        self.targets = torch.randint(0, vocab, (rows,), device=gpu, generator=g)
        self.targets[0] = -100
        if rows > 1:
            used = self.tokens[self.rows[1] if table else 1].clamp(min=0)
            self.targets[1] = used[0]  # a target among the kept tokens
        self.g_ce, self.g_kl = normal(rows), normal(rows)
        self.temperature, self.tail = temperature, "bucket"

    def oracle(self):
        at = self.rows.cpu().numpy() if self.rows is not None else slice(None)
        args = (self.x.double().cpu().numpy(), self.targets.cpu().numpy(), self.tokens.cpu().numpy()[at],
                self.logprobs.double().cpu().numpy()[at])
        more = (self.tail, self.temperature)
        return O.forward(*args, *more), O.grad(*args, self.g_ce.double().cpu().numpy(), self.g_kl.double().cpu().numpy(),
                                               *more)

    def calls(self):
        more = dict(teacher_rows=self.rows, tail=self.tail, temperature=self.temperature, return_argmax=True)
        leaf = self.x.detach().requires_grad_()
        ce, kl, accept, amax = topk_distill_from_logits(leaf, self.targets, self.tokens, self.logprobs, **more)
        (dx,) = torch.autograd.grad([ce, kl], leaf, [self.g_ce, self.g_kl])
        yield "autograd", ce, kl, accept, amax, dx
        ce, kl, accept, dx, amax = topk_distill_fused_grad(self.x, self.targets, self.tokens, self.logprobs,
                                                           ce_weights=self.g_ce, kl_weights=self.g_kl, **more)
        yield "fused", ce, kl, accept, amax, dx

    def check(self):
        (ce, kl, accept, amax), (grad, size) = self.oracle()
        for what, *got in self.calls():
            with np.errstate(invalid="ignore"):
                _close(got[0], ce, STEPS + 4 * U * np.abs(ce), what + " ce")
                _close(got[1], kl, 3 * STEPS * (1 + np.abs(kl)), what + " kl")
            _close(got[2], accept, 2 * STEPS, what + " accept")
            assert np.array_equal(got[3].cpu().numpy(), amax), what
            assert got[4].dtype == self.x.dtype
            _close(got[4], grad, HALF[self.x.dtype] * np.abs(grad) + 3 * STEPS * size + TINY[self.x.dtype],
                   what + " grad")


# one logit, edges of chunks, of a wave's and a workgroup's rows, of the shapes of the one-pass kernel
# (2048, 8192, 32768, 81920, 163840 logits of 16 bits, half as many of fp32), and past them
VOCABS = [1, 2, 7, 9, 300, 1023, 1025, 2048, 2057, 4097, 8193, 16385, 32000, 32777, 50021, 81929, 151936, 163849]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabularies(gpu, vocab, dtype):
    case = Case(gpu, 4, vocab, min(vocab, 19), dtype, vocab)
    case.check()
    case.tail = "renormalize"
    case.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [400, 9001, 32000])
@pytest.mark.parametrize("temperature", [0.5, 3.0])
@pytest.mark.parametrize("kept", [1, 64, 65, 128])
def test_temperatures_and_kept(gpu, vocab, dtype, temperature, kept):
    case = Case(gpu, 5, vocab, kept, dtype, kept, table=3, temperature=temperature)
    case.check()
    case.tail = "renormalize"
    case.check()


@pytest.mark.parametrize("rows", [1, 17, 600])
def test_row_counts(gpu, rows):
    Case(gpu, rows, 10007, 20, torch.bfloat16, rows).check()
    Case(gpu, rows, 10007, 20, torch.bfloat16, rows, table=max(1, rows // 3)).check()


def test_largest_vocabulary(gpu):
    Case(gpu, 2, 524288, 128, torch.float32, 5).check()
    with pytest.raises(NotImplementedError, match="524288"):
        Case(gpu, 2, 524289, 4, torch.float32, 5).check()


def test_many_long_rows(gpu):
    Case(gpu, 270, 90001, 32, torch.float32, 6).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,stride", [(1, 1000), (3, 1003), (0, 1001), (5, 4100)])
def test_strides_and_alignment(gpu, dtype, offset, stride):
    vocab, n = 997, 6
    case = Case(gpu, n, vocab, 9, dtype, 11)
    buffer = torch.zeros(offset + n * stride, dtype=dtype, device=gpu)
    view = buffer[offset:].view(n, stride)[:, :vocab]
    view.copy_(case.x)
    case.x = view
    case.check()
    # in place: the rows become the gradient, the columns behind them stay
    buffer[offset:].view(n, stride)[:, vocab:] = 7
    _, (grad, size) = case.oracle()
    out = topk_distill_fused_grad(view, case.targets, case.tokens, case.logprobs, ce_weights=case.g_ce,
                                  kl_weights=case.g_kl, in_place=True)
    assert out[3].data_ptr() == view.data_ptr()
    _close(view, grad, HALF[dtype] * np.abs(grad) + 3 * STEPS * size + TINY[dtype], "in place")
    assert (buffer[:offset] == 0).all() and (buffer[offset:].view(n, stride)[:, vocab:] == 7).all()


def test_in_place_of_rows_read_twice(gpu):
    case = Case(gpu, 3, 170001, 40, torch.bfloat16, 12)
    _, (grad, size) = case.oracle()
    topk_distill_fused_grad(case.x, case.targets, case.tokens, case.logprobs, ce_weights=case.g_ce,
                            kl_weights=case.g_kl, in_place=True)
    _close(case.x, grad, HALF[torch.bfloat16] * np.abs(grad) + 3 * STEPS * size + 1e-37, "in place")
    with pytest.raises(ValueError, match="in_place"):
        topk_distill_fused_grad(case.x[:, ::2], None, case.tokens, case.logprobs, kl_weights=case.g_kl, in_place=True)


def test_shapes_and_types_of_arguments(gpu):
    case = Case(gpu, 24, 300, 8, torch.bfloat16, 13)
    args = (case.targets, case.tokens, case.logprobs)
    want = topk_distill_from_logits(case.x, *args, return_argmax=True)
    for got in (topk_distill_from_logits(case.x.view(2, 3, 4, 300), *args, return_argmax=True),
                topk_distill_from_logits(case.x.view(2, 3, 4, 300), case.targets.view(2, 3, 4),
                                         case.tokens.view(2, 3, 4, 8), case.logprobs.view(2, 3, 4, 8), return_argmax=True),
                topk_distill_from_logits(case.x, case.targets, case.tokens.int(), case.logprobs, return_argmax=True),
                topk_distill_from_logits(case.x.t().contiguous().t(), case.targets, case.tokens.t().contiguous().t(),
                                         case.logprobs, return_argmax=True)):
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(-1), b)
    assert topk_distill_from_logits(case.x.view(2, 12, 300), *args)[0].shape == (2, 12)
    none = topk_distill_from_logits(case.x, None, case.tokens, case.logprobs, temperature=2.0)
    assert none[0] is None and len(none) == 3
    # no targets: the divergence's gradient alone; unused losses cost nothing
    leaf = case.x.detach().requires_grad_()
    (a,) = torch.autograd.grad(topk_distill_from_logits(leaf, None, case.tokens, case.logprobs)[1].sum(), leaf)
    (b,) = torch.autograd.grad(topk_distill_from_logits(leaf, *args)[1].sum(), leaf)
    ones = torch.ones(24, device=gpu)
    c = topk_distill_fused_grad(case.x, None, case.tokens, case.logprobs, kl_weights=ones)[3]
    torch.testing.assert_close(a, b, atol=0, rtol=0)
    torch.testing.assert_close(a, c, atol=1e-6, rtol=2.0 ** -7)  # a step of bf16 where fp32 differs
    (ce_only,) = torch.autograd.grad(topk_distill_from_logits(leaf, *args)[0].sum(), leaf)
    assert ce_only.isfinite().all() and (ce_only[0] == 0).all()
    empty = topk_distill_from_logits(case.x[:0], case.targets[:0], case.tokens[:0], case.logprobs[:0])
    assert empty[1].shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 2500, 40000])
def test_masks(gpu, dtype, vocab):
    """Tokens without probability among the kept and outside, a tail of nothing, rows of nothing."""
    case = Case(gpu, 9, vocab, 10, dtype, 21, fewer=False)
    x, low = case.x, torch.finfo(dtype).min
    case.targets.fill_(int(vocab // 2))
    case.targets[7] = -100
    ordinary = torch.ones(vocab, dtype=torch.bool, device=gpu)
    ordinary[case.tokens[0]] = ordinary[vocab // 2] = False
    x[0, ordinary] = -float("inf")                  # the tail is the target at most
    x[1, case.tokens[1, :4]] = -float("inf")        # kept tokens the student has no probability for
    x[2] = -float("inf")
    x[3, ordinary] = low
    x[4] = low
    outside = torch.ones(vocab, dtype=torch.bool, device=gpu)
    outside[case.tokens[5]] = False
    x[5, outside] = -float("inf")                   # no tail
    x[6, case.tokens[6]] += 60                      # hardly a tail
    x[7] = -float("inf")
    x[8, case.tokens[8]] = -float("inf")            # nothing but the tail
    case.logprobs[6] = torch.log_softmax(case.logprobs[6], -1) - 1e-3
    case.check()
    case.tail = "renormalize"
    case.check()


def test_confident_teachers_and_students(gpu):
    """Teachers whose kept mass is 1 up to rounding or nearly so, students that agree and that do not."""
    case = Case(gpu, 6, 32000, 16, torch.float32, 31, fewer=False)
    for i, rest in enumerate((0.0, 1e-7, 3e-6, 1e-4, 0.3, 1.0 - 1e-6)):
        case.logprobs[i] = torch.log(torch.softmax(case.logprobs[i].double(), -1) * (1 - rest)).float()
    case.x[::2].scatter_(1, case.tokens[::2], case.logprobs[::2] + 20)
    case.check()


def test_all_tokens_kept_and_nothing_kept(gpu):
    case = Case(gpu, 4, 128, 128, torch.bfloat16, 41, fewer=False)
    case.check()
    case.tokens[:] = -1
    case.logprobs[:] = float("nan")  # unused slots are not read
    for tail in ("bucket", "renormalize"):
        case.tail = tail
        case.check()
    case.g_ce.zero_()
    for _, ce, kl, accept, amax, dx in case.calls():
        assert (kl == 0).all() and (accept == 0).all() and (dx == 0).all()


def test_ties_and_nan(gpu):
    case = Case(gpu, 6, 5000, 12, torch.bfloat16, 51, fewer=False)
    case.x[0] = 2.0                                        # argmax 0
    case.x[1, case.tokens[1, 3]] = case.x[1, 77] = 50.0    # a kept token ties with one outside
    case.x[2, [9, 4000]] = 60.0
    case.check()
    case.x[3, 123] = case.x[3, 99] = float("nan")
    case.x[4, 55] = float("inf")
    case.x[5, case.tokens[5, 2]] = float("nan")
    for _, ce, kl, accept, amax, dx in case.calls():
        assert kl[3:].isnan().all() and accept[3:].isnan().all() and dx[3:].isnan().all()
        assert amax[3:].tolist() == [99, 55, int(case.tokens[5, 2])] and dx[:3].isfinite().all()


@pytest.mark.parametrize("vocab", [500, 40000])
@pytest.mark.parametrize("what", ["token", "negative", "twice", "row", "target"])
def test_bad_indices(gpu, vocab, what):
    case = Case(gpu, 4, vocab, 6, torch.bfloat16, 61, table=4, fewer=False)
    case.rows = torch.arange(4, device=gpu)
    case.targets[:] = 3
    if what == "token":
        case.tokens[2, 5], message = vocab, "teacher token out of range"
    elif what == "negative":
        case.tokens[2, 0], message = -2, "teacher token out of range"
    elif what == "twice":
        case.tokens[2, 4], message = case.tokens[2, 1], "teacher token repeated"
    elif what == "row":
        case.rows[2], message = 4, "teacher index out of range"
    else:
        case.targets[2], message = vocab, "cross-entropy target out of range"
    args = (case.targets, case.tokens, case.logprobs)
    more = {"teacher_rows": case.rows}
    with pytest.raises(ValueError, match=message):
        topk_distill_from_logits(case.x, *args, **more)
    leaf = case.x.clone().requires_grad_()
    with torch.no_grad(), pytest.raises(ValueError, match=message):
        topk_distill_from_logits(leaf, *args, **more)
    ce, kl, accept = topk_distill_from_logits(leaf, *args, **more)
    with pytest.raises(ValueError, match=message):
        (ce + kl).sum().backward()
    weights = {"ce_weights": torch.ones(4, device=gpu), "kl_weights": torch.ones(4, device=gpu)}
    with pytest.raises(ValueError, match=message):
        topk_distill_fused_grad(case.x, *args, **weights, **more)
    ce, kl, accept = topk_distill_from_logits(leaf, *args, check_indices=False, **more)
    (dx,) = torch.autograd.grad((ce + kl).sum(), leaf)
    fused = topk_distill_fused_grad(case.x, *args, check_indices=False, **weights, **more)
    for c, k, d in ((ce, kl, dx), (fused[0], fused[1], fused[3])):
        assert d[2].isnan().all() and d[[0, 1, 3]].isfinite().all()
        assert c[2].isnan() and c[[0, 1, 3]].isfinite().all() and k[[0, 1, 3]].isfinite().all()
        assert k[2].isnan() == (what != "target")


def test_offsets_past_32_bits(gpu):
    """The last rows of a buffer of more than 2^31 elements, in one pass and in place."""
    rows, vocab = 34000, 65536
    case = Case(gpu, 3, vocab, 8, torch.bfloat16, 71)
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=gpu)
    x[-3:] = case.x
    index = torch.zeros(rows, dtype=torch.int64, device=gpu)
    index[-3:] = torch.arange(3, device=gpu)
    targets = torch.zeros(rows, dtype=torch.int64, device=gpu)
    targets[-3:] = case.targets
    w_ce, w_kl = torch.zeros(rows, device=gpu), torch.zeros(rows, device=gpu)
    w_ce[-3:], w_kl[-3:] = case.g_ce, case.g_kl
    topk_distill_fused_grad(x, targets, case.tokens, case.logprobs, ce_weights=w_ce, kl_weights=w_kl,
                            teacher_rows=index, in_place=True)
    _, (grad, size) = case.oracle()
    _close(x[-3:], grad, HALF[torch.bfloat16] * np.abs(grad) + 3 * STEPS * size + 1e-37, "grad")
    assert (x[:5] == 0).all()


@pytest.mark.parametrize("vocab,rows", [(700, 4), (40000, 3)])
def test_graph_replays(gpu, vocab, rows):
    """Forward + backward and the one-pass call captured once; every replay equals the eager call, with
    eager work between and after the inputs change in place."""
    case = Case(gpu, rows, vocab, 10, torch.bfloat16, 81)

    def step(x):
        leaf = x.detach().requires_grad_()
        args = (case.targets, case.tokens, case.logprobs)
        ce, kl, accept = topk_distill_from_logits(leaf, *args)
        (dx,) = torch.autograd.grad([ce, kl], leaf, [case.g_ce, case.g_kl])
        fused = topk_distill_fused_grad(x, *args, ce_weights=case.g_ce, kl_weights=case.g_kl, return_argmax=True)
        return [t.detach() for t in (ce, kl, accept, dx, *fused)]

    static = case.x.clone()
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
        fresh = Case(gpu, rows, vocab, 10, torch.bfloat16, 90 + i).x
        static.copy_(fresh)
        graph.replay()
        want = step(fresh)
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_streams_and_repeats(gpu):
    case = Case(gpu, 40, 20000, 50, torch.float16, 91)
    args = (case.x, case.targets, case.tokens, case.logprobs)
    weights = {"ce_weights": case.g_ce, "kl_weights": case.g_kl}
    want = topk_distill_fused_grad(*args, **weights)
    torch.cuda.synchronize()
    results = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            results += [topk_distill_fused_grad(*args, check_indices=False, **weights) for _ in range(3)]
    torch.cuda.synchronize()
    for got in results:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_teacher_of_token_logprobs(gpu):
    """The two operators as they are used together: a teacher's pass writes the cache, the student trains
    against it; with the teacher's own logits nothing diverges."""
    g = torch.Generator(device=gpu).manual_seed(95)
    teacher = (torch.randn(64, 9000, device=gpu, generator=g) * 3).to(torch.bfloat16)
    for temperature in (1.0, 2.0):
        cache = token_logprobs(teacher, top_k=32, temperature=temperature)
        assert cache.logprobs is None
        leaf = teacher.detach().requires_grad_()
        for tail in ("bucket", "renormalize"):
            _, kl, accept = topk_distill_from_logits(leaf, None, cache.top_indices, cache.top_logprobs, tail=tail,
                                                     temperature=temperature)
            (dx,) = torch.autograd.grad(kl.sum(), leaf)
            if tail == "bucket":
                # log q and log p are off by STEPS + 4 u |logp| each, |logp| <= 40 here; so are the masses
                bound = 2 * (STEPS + 4 * U * 40)
                assert kl.abs().max() <= 2 * bound and (1 - accept).abs().max() <= 2 * bound
                assert dx.float().abs().max() <= 2 * bound
            else:
                mass = cache.top_logprobs.double().exp().sum(-1)
                torch.testing.assert_close(kl.double(), -torch.log(mass), atol=4 * STEPS, rtol=4 * STEPS)
        # in any order, through a table
        order = torch.randperm(64, device=gpu, generator=g)
        back = torch.empty_like(order)
        back[order] = torch.arange(64, device=gpu)
        again = topk_distill_from_logits(teacher, None, cache.top_indices[order].flip(-1).int(),
                                         cache.top_logprobs[order].flip(-1), teacher_rows=back, temperature=temperature)
        want = topk_distill_from_logits(teacher, None, cache.top_indices, cache.top_logprobs, temperature=temperature)
        torch.testing.assert_close(again[1], want[1], atol=6 * STEPS, rtol=0)


def test_saved_tensors_that_move(gpu):
    """Saved tensors kept on the host between forward and backward, logits or a teacher changed in between."""
    case = Case(gpu, 6, 3000, 9, torch.bfloat16, 97, table=4)
    more = {"teacher_rows": case.rows}

    def grad():
        leaf = case.x.clone().requires_grad_()
        ce, kl, _ = topk_distill_from_logits(leaf, case.targets, case.tokens, case.logprobs, **more)
        torch.empty(64, 3000, device=gpu).fill_(9)
        return torch.autograd.grad([ce, kl], leaf, [case.g_ce, case.g_kl])[0]

    want = grad()
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(grad(), want)
    leaf = case.x.clone().requires_grad_()
    _, kl, _ = topk_distill_from_logits(leaf, case.targets, case.tokens, case.logprobs, **more)
    case.logprobs.sub_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kl.sum().backward()


def test_more_rows_than_a_grid_is_wide(gpu):
    """2^21 workgroups are one line of the grid: rows past them equal the same rows alone."""
    rows, vocab = 2 ** 21 + 6, 9
    tail = Case(gpu, 6, vocab, 4, torch.float32, 99)
    x = torch.zeros(rows, vocab, device=gpu)
    x[-6:] = tail.x
    index = torch.zeros(rows, dtype=torch.int64, device=gpu)
    index[-6:] = torch.arange(6, device=gpu)
    targets = torch.zeros(rows, dtype=torch.int64, device=gpu)
    targets[-6:] = tail.targets
    weights = torch.zeros(2, rows, device=gpu)
    weights[0, -6:], weights[1, -6:] = tail.g_ce, tail.g_kl
    leaf = x.requires_grad_()
    ce, kl, accept = topk_distill_from_logits(leaf, targets, tail.tokens, tail.logprobs, teacher_rows=index)
    (dx,) = torch.autograd.grad([ce, kl], leaf, [weights[0], weights[1]])
    fused = topk_distill_fused_grad(x.detach(), targets, tail.tokens, tail.logprobs, ce_weights=weights[0],
                                    kl_weights=weights[1], teacher_rows=index)
    (r_ce, r_kl, r_accept, _), (grad, size) = tail.oracle()
    for got in ((ce, kl, accept, dx), fused):
        _close(got[0][-6:], r_ce, STEPS + 4 * U * np.abs(r_ce), "ce")
        _close(got[1][-6:], r_kl, 3 * STEPS * (1 + np.abs(r_kl)), "kl")
        _close(got[2][-6:], r_accept, 2 * STEPS, "accept")
        _close(got[3][-6:], grad, HALF[torch.float32] * np.abs(grad) + 3 * STEPS * size + 1e-37, "grad")
        assert (got[3][:-6] == 0).all()


def test_in_place_is_seen_by_autograd(gpu):
    """A graph that kept the logits does not use the gradient that has taken their place."""
    case = Case(gpu, 4, 500, 5, torch.float32, 101)
    leaf = case.x.clone().requires_grad_()
    logits = leaf * 1.0
    square = (logits * logits).sum()
    topk_distill_fused_grad(logits, case.targets, case.tokens, case.logprobs, ce_weights=case.g_ce,
                            kl_weights=case.g_kl, in_place=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.backward()
    with torch.inference_mode():  # no graph, no versions
        x = case.x.clone()
        out = topk_distill_fused_grad(x, case.targets, case.tokens, case.logprobs, ce_weights=case.g_ce,
                                      kl_weights=case.g_kl, in_place=True)
        assert out[3].data_ptr() == x.data_ptr() and torch.equal(x, logits.detach())
        assert torch.equal(topk_distill_from_logits(case.x, case.targets, case.tokens, case.logprobs)[1], out[1])
        assert token_logprobs(case.x, top_k=3).top_indices.shape == (4, 3)


@pytest.mark.parametrize("token_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("kept", [1, 2, 63, 64, 65, 128])
def test_the_check_ahead_of_the_pass_finds_what_the_pass_finds(gpu, monkeypatch, kept, token_dtype):
    """The kernel that checks indices alone reports the words that the logits' pass reports, for one bad
    row at either end and between, and none for tokens that only share their lower bits."""
    from aspec_amd import _launch

    rows, vocab, table = 7, 70000, 5
    case = Case(gpu, rows, vocab, kept, torch.bfloat16, 71, table=table, fewer=False)
    weights = {"ce_weights": torch.ones(rows, device=gpu), "kl_weights": torch.ones(rows, device=gpu)}

    def verdicts(targets, tokens, where):
        found = []
        for limit in (0, 1 << 62):
            monkeypatch.setattr(_launch, "CHECK_FIRST_BYTES", limit)
            for entry, more in ((topk_distill_from_logits, {}), (topk_distill_fused_grad, weights)):
                try:
                    out = entry(case.x, targets, tokens, case.logprobs, teacher_rows=where, **more)
                    found.append([v.isnan().any().item() for v in out])
                except ValueError as e:
                    found.append(str(e))
        assert found[0] == found[2] and found[1] == found[3]
        return found[0]

    targets = torch.arange(rows, device=gpu)
    where = torch.arange(rows, device=gpu) % table
    tokens = torch.stack([torch.randperm(vocab, device=gpu)[:kept] for _ in range(table)])
    if kept > 1:
        tokens[0, :2] = torch.tensor([5, 5 + (1 << 15)], device=gpu)  # alike in the lower 15 bits
        tokens[0, 2:] = torch.arange(100, 100 + kept - 2, device=gpu)
    tokens = tokens.to(token_dtype)
    assert verdicts(targets, tokens, where) == [False] * 3
    unused = tokens.clone()
    unused[:, kept // 2:] = -1
    assert verdicts(targets, unused, where) == [False] * 3
    for row in (0, 2, 4):
        for slot in {0, kept // 2, kept - 1}:
            for bad in (vocab, -2, 2**31 - 1):
                changed = tokens.clone()
                changed[row, slot] = bad
                assert "teacher token out of range" in verdicts(targets, changed, where)
            if slot:
                changed = tokens.clone()
                changed[row, slot] = changed[row, slot - 1]
                assert "teacher token repeated" in verdicts(targets, changed, where)
    if kept > 1:
        changed = tokens.clone()
        changed[3, kept - 1] = changed[3, 0]
        assert "teacher token repeated" in verdicts(targets, changed, where)
        # a table row that no row addresses may hold anything
        assert verdicts(targets, changed, where.clamp(max=2)) == [False] * 3
    for row in (0, 3, rows - 1):
        for bad in (-1, vocab, 2**40):
            changed = targets.clone()
            changed[row] = bad
            assert "cross-entropy target out of range" in verdicts(changed, tokens, where)
        for bad in (-1, table, 2**40):
            changed = where.clone()
            changed[row] = bad
            assert "teacher index out of range" in verdicts(targets, tokens, changed)


def test_the_check_ahead_of_the_pass_is_taken_for_large_calls(gpu):
    """Large enough that the check runs on its own: the error comes before the call returns, and the
    results of good indices are the small calls'."""
    rows, vocab = 1100, 16000
    case = Case(gpu, rows, vocab, 3, torch.bfloat16, 72, fewer=False)
    args = (case.targets, case.tokens, case.logprobs)
    from aspec_amd import _launch

    assert case.x.numel() * 2 >= _launch.CHECK_FIRST_BYTES
    kl = topk_distill_from_logits(case.x, *args)[1]
    small = topk_distill_from_logits(case.x[:40], case.targets[:40], case.tokens[:40], case.logprobs[:40])[1]
    unchecked = topk_distill_from_logits(case.x, *args, check_indices=False)[1]
    assert torch.equal(kl, unchecked)
    torch.testing.assert_close(kl[:40], small, rtol=1e-4, atol=1e-5)
    case.tokens[rows - 1, 2] = vocab
    with pytest.raises(ValueError, match="teacher token out of range"):
        topk_distill_from_logits(case.x, *args)
    with pytest.raises(ValueError, match="teacher token out of range"):
        topk_distill_fused_grad(case.x, *args, ce_weights=torch.ones(rows, device=gpu), kl_weights=torch.ones(rows, device=gpu))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [3001, 10240, 16777, 20000, 33000, 36001, 65537, 81919, 100003, 123457])
def test_rows_between_the_shapes(gpu, vocab, dtype):
    """Rows that leave places of a workgroup empty, from no wave's chunk to most of them, with as many
    kept tokens as fit, at temperature 1 and another."""
    case = Case(gpu, 3, vocab, 128, dtype, vocab, temperature=0.8)
    case.check()
    Case(gpu, 3, vocab, 2, dtype, vocab + 1).check()
    wide = torch.randn(3, vocab + 5, device=gpu, generator=torch.Generator(device=gpu).manual_seed(vocab)).to(dtype)
    wide[:, 3:3 + vocab] = case.x
    case.x = wide[:, 3:3 + vocab]  # rows that begin off a chunk's alignment
    case.check()
