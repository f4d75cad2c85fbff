"""Log probabilities, entropy and likeliest tokens against float64 and a stable sort.

fp32 sums: a thread adds up to vocab / 256 exponentials and a row's threads meet in some 16 additions more, each 2^-24 of
the sum; an exponent of y binary places is off by 2^-23 y, which weighs its exponential's share, together the entropy in
bits (17 at most here); the logarithm and the differences round a few times.
"""

from __future__ import annotations

import pytest
import torch

from flextensor_amd import hip

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(gpu, rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=gpu).manual_seed(seed + rows + 5 * vocab)
    x = (torch.randn(rows, vocab, device=gpu, generator=g) * spread).to(dtype)
    return x, torch.randint(0, vocab, (rows,), device=gpu, generator=g)


def _check(got, x, tokens, top):
    given, entropy, best, index = (t.cpu() for t in got)
    x, tokens = x.cpu().double(), tokens.cpu()
    vocab = x.shape[1]
    logp = torch.log_softmax(x, -1)
    unit = 2.0 ** -24 * (vocab / 256 + 16 + 64)
    want = logp.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]
    want = torch.where(tokens < 0, 0.0, torch.where(tokens >= vocab, float("nan"), want))
    _close(given, want, unit)
    share = logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)
    _close(entropy, -share.sum(-1), 2 * unit)
    order = torch.sort(torch.where(x.isnan(), float("inf"), x) + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    rows = ~(x.isnan().any(-1) & (x == float("inf")).any(-1))  # the sort above has NaNs among the infinities
    assert index.dtype == torch.int64 and torch.equal(index[rows], order[rows])
    _close(best, logp.gather(1, index), unit)


def _close(got, want, unit):
    assert got.dtype == torch.float32 and got.shape == want.shape
    same = (got.double() == want) | (got.isnan() & want.isnan())
    near = (got.double() - want).abs() <= unit * (1 + want.abs())
    assert (same | near).all(), (got.double() - want).abs().nan_to_num(0, 0, 0).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 0), (3, 7, 7), (1, 63, 63), (2, 64, 64), (5, 65, 64), (1, 1000, 1), (2, 4095, 20), (7, 4097, 5),
    (1, 32000, 5), (1, 131071, 64), (3, 65537, 20), (40, 32000, 20), (600, 1001, 3), (513, 8193, 64), (1025, 257, 0),
])
def test_rows_match_float64(gpu, dtype, rows, vocab, top):
    print(f"logprobs: {dtype} rows={rows} vocab={vocab} top={top}", flush=True)
    x, tokens = _logits(gpu, rows, vocab, dtype)
    _check(hip.token_logprobs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 600])
def test_orders_that_pass_every_threshold(gpu, dtype, rows):
    """Rising and falling logits, one number throughout, and a few numbers that many share."""
    n = 9001
    x = torch.zeros(rows, n, device=gpu)
    x[0] = torch.linspace(-20, 20, n, device=gpu)
    x[1] = torch.linspace(20, -20, n, device=gpu)
    x[2] = 5.0
    x[3] = torch.randint(0, 4, (n,), device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)).float()
    x[4, 8000:] = 1.0
    x[5, ::3] = -0.0
    x = x.to(dtype)
    tokens = torch.arange(rows, device=gpu) % n
    for top in (1, 20, 64):
        _check(hip.token_logprobs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(10, 5000), (600, 5000), (10, 140000)])
def test_values_that_are_not_finite(gpu, dtype, rows, vocab):
    inf, lowest = float("inf"), torch.finfo(dtype).min
    x, tokens = _logits(gpu, rows, vocab, dtype)
    x[0] = -inf                      # nothing is left
    x[1], x[1, 4321] = -inf, 2.0     # one token is
    x[2] = lowest                    # masked by the lowest number throughout: all alike
    x[3, 1:], x[3, 0] = lowest, 1.0
    x[4, ::2] = -inf
    x[5, 77] = inf
    x[6, 4000] = float("nan")
    x[7, 4000:4003], x[7, 10] = float("nan"), -inf
    x[8] = torch.finfo(dtype).max
    tokens[:10] = torch.tensor([5, 4321, 9, 0, 2, 77, 3, 10, 4999, -1])
    if rows > 10:
        tokens[10], tokens[11], tokens[12] = vocab, vocab + 5, -100
    got = hip.token_logprobs(x, tokens, top=30)
    _check(got, x, tokens, 30)
    assert got[0][0].isnan() and got[1][0].isnan() and got[0][1] == 0 and got[1][1] == 0
    assert got[3][7][:3].tolist() == [4000, 4001, 4002] and got[3][0].tolist() == list(range(30))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_far_logits_keep_their_precision(gpu, dtype):
    x, tokens = _logits(gpu, 4, 3000, dtype, spread=1.0)
    x = (x.float() + torch.tensor([[0.0], [1000.0], [-1000.0], [60000.0]], device=gpu)).to(dtype)
    _check(hip.token_logprobs(x, tokens, top=4), x, tokens, 4)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_of_any_alignment(gpu, dtype):
    for rows, vocab, wide, offset in ((5, 1001, 1003, 1), (3, 40, 77, 3), (700, 333, 1001, 2), (4, 8, 8, 0)):
        held = torch.full((rows + 1, wide), float("nan"), dtype=dtype, device=gpu)
        x, tokens = _logits(gpu, rows, vocab, dtype)
        view = held[:rows, offset: offset + vocab]
        view.copy_(x)
        want = hip.token_logprobs(x, tokens, top=7)
        got = hip.token_logprobs(view, tokens, top=7)
        _check(got, x, tokens, 7)
        assert torch.equal(got[3], want[3])
        _check(hip.token_logprobs(x.t().contiguous().t(), tokens, top=7), x, tokens, 7)
    one, tokens = _logits(gpu, 1, 500, dtype)
    got = hip.token_logprobs(one.expand(6, 500), tokens.expand(6), top=2)
    assert (got[3] == got[3][0]).all() and (got[0] == got[0][0]).all()


def test_refusals_and_empty_calls(gpu):
    x, tokens = _logits(gpu, 4, 100, torch.float32)
    shapes = [t.shape for t in hip.token_logprobs(x[:0], tokens[:0], top=3)]
    assert shapes == [(0,), (0,), (0, 3), (0, 3)]
    assert hip.token_logprobs(x, tokens)[2].shape == (4, 0)
    for bad in (lambda: hip.token_logprobs(x, tokens, top=65), lambda: hip.token_logprobs(x, tokens, top=-1),
                lambda: hip.token_logprobs(x[:, :9], tokens, top=10), lambda: hip.token_logprobs(x, tokens[:3]),
                lambda: hip.token_logprobs(x[0], tokens), lambda: hip.token_logprobs(x[:, :0], tokens),
                lambda: hip.token_logprobs(x, tokens.cpu()), lambda: hip.token_logprobs(x.cpu(), tokens.cpu()),
                lambda: hip.token_logprobs(x.clone().requires_grad_(), tokens)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hip.token_logprobs(x.double(), tokens), lambda: hip.token_logprobs(x, tokens.int())):
        with pytest.raises(TypeError):
            bad()
