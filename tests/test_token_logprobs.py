"""CPU checks of the token log-probabilities: the fp64 oracle against closed forms, torch and
differences, and the refusals of the Python call and the C entries."""

import ctypes

import numpy as np
import pytest
import torch

from aspec_amd import _lib, token_logprobs
from oracle import token_logprobs as O


def test_oracle_against_torch_and_closed_forms():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 33, generator=g, dtype=torch.float64) * 3
    ids = torch.tensor([0, 32, 5, -100, 7, 7, 1])
    lp, h, top, order = O.forward(x.numpy(), ids.numpy(), 4, 0.7)
    ref = torch.log_softmax(x / 0.7, -1)
    want = torch.where(ids < 0, 0.0, ref.gather(1, ids.clamp(min=0)[:, None])[:, 0])
    np.testing.assert_allclose(lp, want, rtol=1e-13)
    np.testing.assert_allclose(h, torch.distributions.Categorical(logits=x / 0.7).entropy(), rtol=1e-13)
    np.testing.assert_allclose(top, ref.sort(-1, descending=True).values[:, :4], rtol=1e-13)
    # uniform over the unmasked tokens; ties by index
    x = np.full((1, 12), -np.inf)
    x[0, 3:11] = 2.5
    lp, h, top, order = O.forward(x, np.array([4]), 10)
    assert abs(lp[0] + np.log(8)) < 1e-15 and abs(h[0] - np.log(8)) < 1e-15
    assert order[0].tolist() == [3, 4, 5, 6, 7, 8, 9, 10, 0, 1] and np.isneginf(top[0, 8:]).all()
    # a row of nothing
    lp, h, top, order = O.forward(np.full((1, 3), -np.inf), np.array([1]), 3)
    assert np.isneginf(lp[0]) and h[0] == 0 and order[0].tolist() == [0, 1, 2]
    # -0 and +0 tie, NaN first
    assert O.top_order(np.array([[-0.0, 0.0, 1.0]]))[0].tolist() == [2, 0, 1]
    assert O.top_order(np.array([[1.0, np.nan, np.inf]]))[0].tolist() == [1, 2, 0]


def test_oracle_gradient_against_differences():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(3, 9)) * 2
    ids, k, temperature = np.array([2, -100, 8]), 3, 1.7
    gl, gh, gt = rng.normal(size=3), rng.normal(size=3), rng.normal(size=(3, k))

    def loss(x):
        lp, h, top, _ = O.forward(x, ids, k, temperature)
        return (gl * lp).sum() + (gh * h).sum() + (gt * top).sum()

    got = O.grad(x, ids, gl, gh, gt, k, temperature)
    step = 1e-6
    for i, j in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i, j] += step
        down[i, j] -= step
        assert abs((loss(up) - loss(down)) / (2 * step) - got[i, j]) < 1e-8


def test_refusals_of_the_call():
    x = torch.randn(2, 5)
    with pytest.raises(ValueError, match="CUDA logits"):
        token_logprobs(x, torch.tensor([0, 1]))
    for temperature in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            token_logprobs(x, temperature=temperature)
    for top_k in (-1, 1.5, True):
        with pytest.raises(ValueError, match="top_k"):
            token_logprobs(x, top_k=top_k)
    for ids in (torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0, 1, 2]), torch.tensor([[0, 1, 2]])):
        with pytest.raises(ValueError, match="one int64 token per logit row"):
            token_logprobs(x, ids)


def test_refusals_of_the_c_entries():
    lib = _lib.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call below fails its checks

    def fwd(dtype=4, rows=2, vocab=100, stride=100, temperature=1.0, top_k=5, logits=fake, ids=fake, logprobs=fake,
            top=fake, workspace=None):
        _lib.check(lib.aspec_token_logprobs_fwd(logits, dtype, rows, vocab, stride, ids, -100, temperature, top_k,
                                                logprobs, fake, top, top, fake, workspace, None, None))

    def bwd(grad=fake, top_indices=fake, ids=fake, stride=100, grad_stride=100, logits=fake):
        _lib.check(lib.aspec_token_logprobs_bwd(logits, 4, 2, 100, stride, ids, -100, 1.0, 5, top_indices, fake, fake,
                                                fake, fake, grad, grad_stride, None))

    with pytest.raises(NotImplementedError, match="bf16, fp16 or fp32"):
        fwd(dtype=1)
    for bad in ({"rows": -1}, {"vocab": 0}, {"stride": 99}):
        with pytest.raises(ValueError, match="at least as far apart"):
            fwd(**bad)
    with pytest.raises(NotImplementedError, match="524288"):
        fwd(vocab=524289, stride=524289)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-45, 3e38):
        with pytest.raises(ValueError, match="temperature"):
            fwd(temperature=temperature)
    for top_k in (-1, 101):
        with pytest.raises(ValueError, match="top_k"):
            fwd(top_k=top_k)
    with pytest.raises(NotImplementedError, match="128"):
        fwd(vocab=1000, stride=1000, top_k=129)
    # (the last one: a row cut into parts without the workspace that joins them)
    for bad in ({"logits": None}, {"logprobs": None}, {"top": None}, {"rows": 1, "vocab": 151936, "stride": 151936}):
        with pytest.raises(ValueError, match="null pointer"):
            fwd(**bad)
    for bad in ({"logits": None}, {"grad": None}, {"top_indices": None}, {"ids": None}):
        with pytest.raises(ValueError, match="null pointer"):
            bwd(**bad)
    for bad in ({"stride": 99}, {"grad_stride": 99}):
        with pytest.raises(ValueError, match="at least as far apart"):
            bwd(**bad)
    with pytest.raises(ValueError, match="in place"):
        bwd(grad=ctypes.c_void_p(8192), logits=ctypes.c_void_p(8192))
    size = ctypes.c_size_t(1)
    assert lib.aspec_token_logprobs_workspace_bytes(4, 4096, 32000, 64, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.aspec_token_logprobs_workspace_bytes(4, 1, 151936, 20, ctypes.byref(size)) == 0 and size.value > 0
    fwd(rows=0)  # nothing to do


def test_refusals_of_the_check_entry():
    lib = _lib.load()
    fake = ctypes.c_void_p(4096)  # never dereferenced: every call fails its checks, or has no rows

    def check(ids=fake, rows=2, vocab=100, words=fake):
        _lib.check(lib.aspec_token_logprobs_check(ids, rows, vocab, -100, words, None))

    for error, match, bad in ((ValueError, "at least as far apart", {"rows": -1}),
                              (ValueError, "at least as far apart", {"vocab": 0}),
                              (NotImplementedError, "524288", {"vocab": 524289}),
                              (ValueError, "null pointer", {"ids": None}), (ValueError, "null pointer", {"words": None})):
        with pytest.raises(error, match=match):
            check(**bad)
    check(rows=0)
