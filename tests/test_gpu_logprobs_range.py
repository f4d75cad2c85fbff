"""Log probabilities over the range of finite logits: rows masked by a large finite number, rows whose largest logits are
far from 0, and rows that cross from far to near.

The tolerance is the one of ordinary rows: a logit's difference from the row's maximum rounds once whatever their size.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_logprobs import TYPES, _check, _logits

from flextensor_amd import hip

pytestmark = pytest.mark.gpu

MASKS = [-1e4, -6e4, -1e5, -1e9, -1e10, -1e12, -1e20, -1e25, -1e30, -1e32, -3e38]
MAXIMA = [1e3, 6e4, 1e5, 1e6, 1.5e7, 1e8, 1e9, 1.2e10, 1e20, 1e30, 3e38]


def _of(values, dtype):
    return [v for v in values if abs(v) < torch.finfo(dtype).max]


def _run(x, tokens, rows, top):
    """The cases, and as many rows of them as make the other launches."""
    x, tokens = x.repeat(-(-rows // len(x)), 1)[:rows].contiguous(), tokens.repeat(-(-rows // len(tokens)))[:rows]
    _check(hip.token_logprobs(x, tokens, top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(66, 5000, 20), (600, 5000, 20), (600, 33000, 0), (66, 140001, 5), (9, 140001, 0)])
def test_rows_masked_by_a_finite_number(gpu, dtype, rows, vocab, top):
    print(f"masked logits: {dtype} rows={rows} vocab={vocab} top={top}", flush=True)
    masks = _of(MASKS, dtype)
    x, tokens = _logits(gpu, 6 * len(masks), vocab, dtype, seed=rows)
    g = torch.Generator(device=gpu).manual_seed(vocab)
    for i, mask in enumerate(masks):
        x[i, : vocab * 3 // 4] = mask                                              # the start
        x[i + len(masks), vocab // 3:] = mask                                      # the end: a padded vocabulary
        at = 2 * len(masks) + i
        keep = x[at, vocab // 2].clone()
        x[at], x[at, vocab // 2] = mask, keep                                      # all but one
        x[i + 3 * len(masks)].masked_fill_(torch.rand(vocab, device=gpu, generator=g) < 0.97, mask)  # most of them
        x[i + 4 * len(masks), ::2] = mask
        x[i + 5 * len(masks)] = mask                                               # all: equally likely
    tokens[::3] = vocab // 2
    _run(x, tokens, rows, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(22, 3, 2), (22, 5000, 20), (600, 5000, 20), (600, 7001, 0), (22, 140001, 5)])
def test_rows_whose_largest_logits_are_far_from_0(gpu, dtype, rows, vocab, top):
    print(f"far logits: {dtype} rows={rows} vocab={vocab} top={top}", flush=True)
    ends = [s * v for v in _of(MAXIMA, dtype) for s in (1, -1)]
    x, tokens = _logits(gpu, len(ends), vocab, dtype, seed=1)
    far = torch.tensor(ends, device=gpu, dtype=torch.float64)[:, None]
    x = (far + x.double()).clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
    if vocab == 3:
        x[:] = far.to(dtype)  # three equal logits
    _run(x, tokens, rows, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 600])
def test_rows_that_cross_from_far_to_near(gpu, dtype, rows):
    """Maxima that rise from the lowest numbers to the largest, and rows around 2^16 on both sides of 0."""
    vocab, most = 40001, torch.finfo(dtype).max
    x = torch.zeros(12, vocab, device=gpu, dtype=torch.float64)
    ramp = torch.linspace(-1, 1, vocab, device=gpu, dtype=torch.float64)
    steps = torch.linspace(0, 1, vocab, device=gpu, dtype=torch.float64)
    for i, size in enumerate((7e4, 1e6, 1e9, 1e30)):
        x[i], x[i + 4] = ramp * size, -ramp * size
    noise = torch.randn(4, vocab, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)).double() * 4
    x[8], x[9] = 65536 + noise[0], -65536 + noise[1]
    x[10] = -(10.0 ** (30 * (1 - steps))) + noise[2]   # from -1e30 up to about 0, a little at a time
    x[11] = -65536 - 8 + 16 * steps + noise[3] * 0.1
    x = x.clamp(-most, most).to(dtype)
    tokens = torch.arange(12, device=gpu) * 3001
    for top in (0, 20):
        _run(x, tokens, rows, top)
