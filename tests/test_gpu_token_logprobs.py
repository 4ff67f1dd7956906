"""Token log-probabilities, entropy, best alternatives and their gradient on the GPU against the fp64
oracle, at the sizes and masks where the kernels' cuts, lists and searches lie.

Tolerances (u = 2^-24, half a step of fp32). The row sum is at most 96 rounded additions deep
(64 + 1 per thread, 6 + 5 joining lanes, waves and parts, each at most u relative, and the factors
that rebase it); an exponent d = (x - m) / temperature carries 4 u |d| from its two products and its
scale, and v_exp_f32 and v_log_f32 one step each: a log-probability is off by at most
u (128 + 4 spread) + 4 u |logp|, a probability by that much relative, where `spread` is |d| of the
terms that matter: e^-60 weighs nothing in fp32, so 60. A gradient is a sum of terms with that
relative error, rounded once to its type."""

import numpy as np
import pytest
import torch

from aspec_amd import token_logprobs
from oracle import token_logprobs as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEPS = U * (128 + 4 * 60)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24, torch.float32: 1e-37}  # below the normal range
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _close(got, ref, tol, what):
    got = got.double().cpu().numpy()
    assert got.shape == ref.shape, what
    same = (got == ref) | (np.isnan(got) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - ref) <= tol))
    assert not bad.any(), (what, np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5])


def check(x, ids, top_k, temperature=1.0, seed=3):
    """Forward and gradient of logits x [n, V] against the oracle."""
    n, vocab = x.shape
    rng = np.random.default_rng(seed)
    gl, gh, gt = (rng.normal(size=s).astype(np.float32) for s in (n, n, (n, top_k)))
    leaf = x.detach().requires_grad_()
    out = token_logprobs(leaf, ids, top_k=top_k, temperature=temperature)
    x64, ids64 = x.detach().double().cpu().numpy(), ids.cpu().numpy()
    lp, h, top, order = O.forward(x64, ids64, top_k, temperature)
    with np.errstate(invalid="ignore"):
        lp_tol, top_tol = STEPS + 4 * U * np.abs(lp), STEPS + 4 * U * np.abs(top)
    _close(out.logprobs.detach(), lp, lp_tol, "logprobs")
    # entropy: sum p |logp| of terms with a relative error STEPS each, and log S
    _close(out.entropy.detach(), h, 2 * STEPS * (1 + np.nan_to_num(h)), "entropy")
    grads = [torch.as_tensor(gl, device=x.device), torch.as_tensor(gh, device=x.device)]
    losses = [out.logprobs, out.entropy]
    if top_k:
        assert np.array_equal(out.top_indices.cpu().numpy(), order)
        _close(out.top_logprobs.detach(), top, top_tol, "top_logprobs")
        losses.append(out.top_logprobs)
        grads.append(torch.as_tensor(gt, device=x.device))
    else:
        assert out.top_logprobs is None and out.top_indices is None
    (dx,) = torch.autograd.grad(losses, leaf, grads)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    ref = O.grad(x64, ids64, gl.astype(np.float64), gh.astype(np.float64), gt.astype(np.float64), top_k, temperature)
    logp = O.log_softmax(x64, temperature)
    p = np.nan_to_num(np.exp(logp))
    size = np.abs(gl)[:, None] * p + np.abs(gh)[:, None] * p * (np.abs(np.where(p > 0, logp, 0.0)) + h[:, None] + 1)
    size += np.abs(gt).sum(axis=-1, keepdims=True) * p
    rows = np.arange(n)
    ok = (ids64 >= 0) & (ids64 < vocab)
    np.add.at(size, (rows[ok], ids64[ok]), np.abs(gl)[ok])
    if top_k:
        np.add.at(size, (rows[:, None], order), np.abs(gt))
    tol = HALF[x.dtype] * np.abs(ref) + 2 * STEPS * np.nan_to_num(size) / temperature + TINY[x.dtype]
    _close(dx, ref, tol, "grad")
    return out


def logits(gpu, n, vocab, dtype, seed, scale=3.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(n, vocab, device=gpu, generator=g) * scale).to(dtype), g


# one logit, less than a chunk, a lone tail, a wave's 2048 (16-bit) or 1024 (fp32) logits and one
# more, a workgroup's 8192 / 4096, rows in parts, and the largest vocabulary
VOCABS = [1, 2, 7, 8, 9, 63, 513, 1023, 1024, 1025, 2048, 2055, 2056, 4097, 8192, 8200, 8201, 32000, 32768, 50021, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabularies(gpu, vocab, dtype):
    n = 5
    x, g = logits(gpu, n, vocab, dtype, vocab)
    ids = torch.tensor([0, vocab - 1, vocab // 2, -100, vocab // 3], device=gpu)
    check(x, ids, min(vocab, 20))
    check(x, ids, min(vocab, 128), temperature=0.6)


@pytest.mark.parametrize("rows", [1, 2, 511, 512, 600])
def test_row_counts(gpu, rows):
    """Few rows share workgroups' parts, many take a workgroup each."""
    x, g = logits(gpu, rows, 10007, torch.bfloat16, rows)
    check(x, torch.randint(0, 10007, (rows,), device=gpu, generator=g), 9)


def test_largest_vocabulary(gpu):
    x, g = logits(gpu, 2, 524288, torch.float32, 5)
    check(x, torch.tensor([524287, 1], device=gpu), 128)
    with pytest.raises(NotImplementedError, match="524288"):
        token_logprobs(torch.zeros(1, 524289, device=gpu))


def test_many_long_rows(gpu):
    """Rows of several of the largest parts, more rows than share a part."""
    x, g = logits(gpu, 300, 70001, torch.bfloat16, 6)
    check(x, torch.randint(0, 70001, (300,), device=gpu, generator=g), 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,stride", [(1, 1000), (3, 1003), (0, 1001), (5, 4100)])
def test_strides_and_alignment(gpu, dtype, offset, stride):
    vocab, n = 997, 6
    buffer, g = logits(gpu, 1, offset + n * stride, dtype, 11)
    x = buffer[0, offset:].view(n, stride)[:, :vocab]
    ids = torch.randint(0, vocab, (n,), device=gpu, generator=g)
    a = check(x, ids, 5)
    b = token_logprobs(x.contiguous(), ids, top_k=5)
    assert torch.equal(a.top_indices, b.top_indices)


def test_leading_dimensions_and_layouts(gpu):
    x, g = logits(gpu, 24, 300, torch.bfloat16, 12)
    ids = torch.randint(0, 300, (24,), device=gpu, generator=g)
    want = token_logprobs(x, ids, top_k=3)
    got = token_logprobs(x.view(2, 3, 4, 300), ids.view(2, 3, 4), top_k=3)
    assert got.logprobs.shape == got.entropy.shape == (2, 3, 4) and got.top_indices.shape == (2, 3, 4, 3)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    columns = x.t().contiguous().t()  # elements a row apart
    for a, b in zip(token_logprobs(columns, ids, top_k=3), want):
        assert torch.equal(a, b)
    leaf = columns.detach().requires_grad_()
    (dx,) = torch.autograd.grad(token_logprobs(leaf, ids).logprobs.sum(), leaf)
    (ref,) = torch.autograd.grad(token_logprobs(x.requires_grad_(), ids).logprobs.sum(), x)
    assert torch.equal(dx, ref)
    # One row, four times: a row at another address is cut elsewhere and summed in another order, so
    # the two results differ by up to twice the error of each.
    wide = x[:1].detach().expand(4, 300)
    torch.testing.assert_close(token_logprobs(wide, ids[:4]).entropy, want.entropy[:1].expand(4), atol=4 * STEPS,
                               rtol=4 * STEPS)
    one = token_logprobs(x[0].detach(), ids[0].reshape(()))
    assert one.logprobs.shape == ()
    torch.testing.assert_close(one.logprobs, want.logprobs[0], atol=2 * STEPS, rtol=8 * U)
    none = token_logprobs(x[:0].detach().requires_grad_(), ids[:0], top_k=4)
    assert none.logprobs.shape == (0,) and none.top_indices.shape == (0, 4)
    assert token_logprobs(x.detach()).logprobs is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 1200, 9000, 40000])
def test_masks(gpu, dtype, vocab):
    """-inf, the type's lowest value and -1e4 in masked places, rows with less than K or nothing left,
    a given token that is masked."""
    x, g = logits(gpu, 8, vocab, dtype, 21 + vocab)
    x[0, vocab // 2:] = -float("inf")
    x[1, 3:] = -float("inf")
    x[2] = -float("inf")
    x[3, 1:] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[5, ::2] = -1e4
    x[6, :vocab - 1] = -float("inf")
    x[7, 0] = torch.finfo(dtype).max
    ids = torch.tensor([vocab - 1, 1, 0, 0, 5, 2, vocab - 1, 0], device=gpu)
    out = check(x, ids, 20)
    assert out.logprobs[0].item() == out.logprobs[2].item() == -float("inf") and out.entropy[2].item() == 0


@pytest.mark.parametrize("vocab", [100, 1500, 9001, 32768, 80000])
@pytest.mark.parametrize("top_k", [1, 20, 128])
def test_ties_and_clusters(gpu, vocab, top_k):
    """Rows whose best tokens are equal, lie side by side or rise to the row's end: lists that overflow."""
    k = min(top_k, vocab)
    x, g = logits(gpu, 8, vocab, torch.bfloat16, 31)
    x[0] = 1.25                                                    # all equal
    x[1] = torch.arange(vocab, device=gpu) * (40.0 / vocab)        # rising
    x[2] = torch.arange(vocab, 0, -1, device=gpu) * (40.0 / vocab)  # falling
    x[3, : vocab // 2] = 9.0                                       # half the row ties
    x[4, vocab // 3: vocab // 3 + min(700, vocab // 3)] = 20.0     # a long run
    x[5] = torch.where(torch.arange(vocab, device=gpu) % 2 == 0, 0.0, -0.0)
    x[6] = torch.randint(0, 3, (vocab,), device=gpu, generator=g).to(torch.bfloat16)
    x[7, :64] += 30
    check(x, torch.randint(0, vocab, (8,), device=gpu, generator=g), k)


@pytest.mark.parametrize("vocab", [50, 3000, 40000])
def test_nan_and_inf(gpu, vocab):
    x, g = logits(gpu, 6, vocab, torch.float32, 41)
    x[0, 7] = float("nan")
    x[1, 9] = float("inf")
    x[2] = float("nan")
    x[3, 11], x[3, 5] = float("inf"), float("nan")
    x[4, vocab // 2:] = float("nan")
    check(x, torch.randint(0, vocab, (6,), device=gpu, generator=g), 30)


def test_confident_and_flat_rows(gpu):
    x, g = logits(gpu, 4, 32000, torch.float32, 51, scale=1e-3)
    x[1, 77] = 40.0
    x[2] *= 1e4
    x[3, 5] = 14.0
    check(x, torch.tensor([0, 77, 1, 5], device=gpu), 8)


def test_bad_tokens(gpu):
    x, g = logits(gpu, 3, 500, torch.bfloat16, 61)
    ids = torch.tensor([3, 500, -1], device=gpu)
    with pytest.raises(ValueError, match="token id out of range"):
        token_logprobs(x, ids)
    with torch.no_grad(), pytest.raises(ValueError, match="token id out of range"):
        token_logprobs(x.clone().requires_grad_(), ids)
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, ids)  # the backward raises
    with pytest.raises(ValueError, match="token id out of range"):
        out.logprobs.sum().backward()
    out = token_logprobs(leaf, ids, check_ids=False)
    assert out.logprobs.isnan().tolist() == [False, True, True] and out.entropy.isfinite().all()
    (dx,) = torch.autograd.grad(out.logprobs.sum(), leaf)
    assert dx[0].isfinite().all() and dx[1:].isnan().all()
    huge = token_logprobs(x, torch.tensor([3, 2 ** 32 + 3, -2 ** 40], device=gpu), check_ids=False)
    assert huge.logprobs.isnan().tolist() == [False, True, True]
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, top_k=501)
    with pytest.raises(ValueError, match="BF16, FP16 or FP32"):
        token_logprobs(x.double())


def test_offsets_past_32_bits(gpu):
    """The last rows of a buffer of more than 2^31 elements equal the same rows alone."""
    rows, vocab = 34000, 65536
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=gpu)
    tail, g = logits(gpu, 3, vocab, torch.bfloat16, 71)
    x[-3:] = tail
    ids = torch.randint(0, vocab, (rows,), device=gpu, generator=g)
    leaf = x.requires_grad_()
    out = token_logprobs(leaf, ids, top_k=2)
    (dx,) = torch.autograd.grad(out.logprobs.sum(), leaf)
    del leaf, x
    want = check(tail, ids[-3:], 2)
    assert torch.equal(out.top_indices[-3:], want.top_indices)
    torch.testing.assert_close(out.logprobs[-3:], want.logprobs, atol=STEPS, rtol=4 * U)
    ref = O.grad(tail.double().cpu().numpy(), ids[-3:].cpu().numpy(), np.ones(3), np.zeros(3), np.zeros((3, 2)), 2)
    torch.testing.assert_close(dx[-3:].double().cpu(), torch.as_tensor(ref), atol=1e-6, rtol=2.0 ** -7)


@pytest.mark.parametrize("vocab,rows", [(700, 4), (40000, 3)])
def test_graph_replays(gpu, vocab, rows):
    """Forward and backward captured once; every replay equals the eager call, with eager work between
    and after the inputs change in place."""
    x, g = logits(gpu, rows, vocab, torch.bfloat16, 81)
    ids = torch.randint(0, vocab, (rows,), device=gpu, generator=g)
    gl = torch.randn(rows, device=gpu, generator=g)

    def step(leaf):
        out = token_logprobs(leaf, ids, top_k=7)
        (dx,) = torch.autograd.grad([out.logprobs, out.entropy], leaf, [gl, gl])
        return *(t.detach() for t in out), dx

    static = x.clone().requires_grad_()
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
        fresh, _ = logits(gpu, rows, vocab, torch.bfloat16, 90 + i)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        want = step(fresh.clone().requires_grad_())
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_streams_and_repeats(gpu):
    """Two streams at once and the same call again give the same bits."""
    x, g = logits(gpu, 40, 20000, torch.float16, 91)
    ids = torch.randint(0, 20000, (40,), device=gpu, generator=g)
    want = token_logprobs(x, ids, top_k=50)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            results += [token_logprobs(x, ids, top_k=50, check_ids=False) for _ in range(3)]
    torch.cuda.synchronize()
    for got in results:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_neighbours_stay_as_they_were(gpu):
    """A view's padding columns are neither read into a result nor written."""
    vocab, stride = 509, 520
    buffer = torch.full((7, stride), float("nan"), dtype=torch.bfloat16, device=gpu)
    x, g = logits(gpu, 7, vocab, torch.bfloat16, 95)
    buffer[:, :vocab] = x
    out = token_logprobs(buffer[:, :vocab], torch.zeros(7, dtype=torch.int64, device=gpu), top_k=20)
    assert out.logprobs.isfinite().all() and int(out.top_indices.max()) < vocab
    assert buffer[:, vocab:].isnan().all() and torch.equal(buffer[:, :vocab], x)


def test_saved_tensors_that_move(gpu):
    """Saved tensors kept on the host between forward and backward, and logits changed in between."""
    x, g = logits(gpu, 6, 3000, torch.bfloat16, 97)
    ids = torch.randint(0, 3000, (6,), device=gpu, generator=g)

    def grad():
        leaf = x.clone().requires_grad_()
        out = token_logprobs(leaf, ids, top_k=4)
        torch.empty(64, 3000, device=gpu).fill_(9)
        return torch.autograd.grad(out.logprobs.sum() + out.top_logprobs.sum(), leaf)[0]

    want = grad()
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(grad(), want)
    leaf = x.clone().requires_grad_()
    twice = leaf * 2
    out = token_logprobs(twice, ids)
    twice.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


def test_more_rows_than_a_grid_is_wide(gpu):
    """2^21 workgroups are one line of the grid: rows past them, small vocabularies."""
    rows, vocab = 2 ** 21 + 5, 8
    x, g = logits(gpu, rows, vocab, torch.bfloat16, 99)
    ids = torch.randint(0, vocab, (rows,), device=gpu, generator=g)
    leaf = x.requires_grad_()
    out = token_logprobs(leaf, ids, top_k=3)
    (dx,) = torch.autograd.grad(out.logprobs.sum(), leaf)
    want = torch.log_softmax(x.detach().double(), -1)
    torch.testing.assert_close(out.logprobs.double(), want.gather(1, ids[:, None])[:, 0], atol=STEPS, rtol=4 * U)
    assert torch.equal(out.top_indices, x.detach().float().sort(dim=-1, descending=True, stable=True).indices[:, :3])
    ref = torch.nn.functional.one_hot(ids, vocab) - want.exp()
    torch.testing.assert_close(dx.double(), ref, atol=4 * STEPS, rtol=2.0 ** -8)


@pytest.mark.parametrize("temperature", [1e-3, 1e-30, 1e30])
def test_extreme_temperatures(gpu, temperature):
    """Nearly all or nearly none of the spread: the largest tokens share everything, or all tokens do."""
    x, g = logits(gpu, 3, 700, torch.float32, 100)
    x[1, 5] = -float("inf")
    x[2, [7, 9]] = 30.0
    out = token_logprobs(x, torch.tensor([0, 5, 9], device=gpu), top_k=4, temperature=temperature)
    if temperature < 1:
        assert out.logprobs[2].item() == pytest.approx(-np.log(2), abs=STEPS)
        assert out.entropy.tolist() == pytest.approx([0.0, 0.0, np.log(2)], abs=2 * STEPS)
    else:
        assert out.logprobs[0].item() == pytest.approx(-np.log(700), abs=2 * STEPS)
        assert out.entropy.tolist() == pytest.approx([np.log(700), np.log(699), np.log(700)], abs=16 * STEPS)
    assert out.logprobs[1].item() == -float("inf")


@pytest.mark.parametrize("row", [0, 255, 256, 1099])
@pytest.mark.parametrize("bad", [-1, 16000, 2**40])
def test_a_bad_id_of_a_large_call_raises_before_it_returns(gpu, row, bad):
    """Such a call checks its tokens in a kernel of their own, ahead of the logits' pass."""
    from aspec_amd import _launch

    x = torch.randn(1100, 16000, device=gpu, dtype=torch.bfloat16)
    assert x.numel() * 2 >= _launch.CHECK_FIRST_BYTES
    ids = torch.arange(1100, device=gpu)
    ids[7] = -100
    good = token_logprobs(x, ids)
    assert torch.equal(good.logprobs, token_logprobs(x, ids, check_ids=False).logprobs)
    ids[row] = bad
    with pytest.raises(ValueError, match="token id out of range"):
        token_logprobs(x, ids)
    assert token_logprobs(x, ids, check_ids=False).logprobs[row].isnan()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab,top_k", [(64, 64), (65, 7), (200, 60), (257, 128), (500, 64), (511, 1), (512, 128),
                                         (1500, 64), (2047, 128), (2049, 128), (4099, 128)])
def test_many_alternatives_of_few_tokens(gpu, vocab, top_k, dtype):
    """Lists much longer than the number of alternatives: the same alternatives, in the same order, for
    random, tied, masked and NaN rows."""
    g = torch.Generator(device=gpu).manual_seed(vocab + top_k)
    x = torch.randn(70, vocab, device=gpu, generator=g)
    x[10:20] = x[10:20].mul(4).round().div(4)  # ties
    x[20:24] = 1.5
    x[24:30, torch.randperm(vocab, device=gpu, generator=g)[vocab // 3:]] = float("-inf")
    x[30, ::7] = float("nan")
    x[31] = float("nan")
    x[32:40] = torch.arange(vocab, device=gpu).float() / 8
    x[40:45] = -x[32:37]
    x[45:50] = torch.finfo(dtype).min
    x[45:50, vocab // 2] = 1.0
    x = x.to(dtype)
    got = token_logprobs(x, top_k=top_k)
    order = O.top_order(x.float().cpu().numpy())[:, :top_k]
    assert np.array_equal(got.top_indices.cpu().numpy(), order)
    few = token_logprobs(x, top_k=1)
    assert torch.equal(got.entropy.nan_to_num(7.0), few.entropy.nan_to_num(7.0))
    assert torch.equal(got.top_logprobs[:, :1].nan_to_num(7.0), few.top_logprobs.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [700, 3001, 10240, 16777, 20000, 36001, 81919, 100003])
def test_rows_between_the_shapes(gpu, vocab, dtype):
    """Rows that leave places of a workgroup empty, from no wave's chunk to most of them."""
    g = torch.Generator(device=gpu).manual_seed(vocab)
    wide = (torch.randn(5, vocab + 5, device=gpu, generator=g) * 3).to(dtype)
    for x in (wide[:, :vocab], wide[:, 3:3 + vocab]):
        ids = torch.tensor([0, vocab - 1, vocab // 2, -100, 1], device=gpu)
        got = token_logprobs(x, ids, top_k=100, temperature=0.8)
        lp, entropy, top, order = O.forward(x.double().cpu().numpy(), ids.cpu().numpy(), 100, 0.8)
        assert np.array_equal(got.top_indices.cpu().numpy(), order)
        _close(got.logprobs, lp, STEPS + 4 * U * np.abs(lp), "logprobs")
        _close(got.entropy, entropy, 2 * STEPS * (1 + entropy), "entropy")
        _close(got.top_logprobs, top, STEPS + 4 * U * np.abs(top), "top_logprobs")
