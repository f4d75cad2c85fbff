"""Places of a tree's nodes that were never written: the sequences of a batch add fewer tokens than the tree has nodes, or
the rows see some of the nodes only. Codes of NaN and scales of NaN there change no bit of the result.

What the rows do see is compared with float64; the tolerance is that of the attention without a tree.
"""

from __future__ import annotations

import pytest
import torch
from test_gpu_kv_cache import BLOCK, FORMATS, TWO_ROUNDINGS, _gen
from test_gpu_kv_tree import _i32, _sets
from test_gpu_kv_tree_dealt import _cache, _dealt, _exact

from flextensor_amd import kv_cache as kvc

pytestmark = pytest.mark.gpu


def _spoil(codes, scales, page, block, first, whole):
    """Tokens `first` on of a block get codes of NaN (the largest int8); with `whole` the block's scales are NaN too."""
    raw = codes.view(torch.uint8)
    d = codes.shape[-1] // BLOCK
    raw[page, 0, :, block].view(-1, d // 16, BLOCK, 16)[:, :, first:] = 127
    raw[page, 1, :, block].view(-1, d, BLOCK)[..., first:] = 127
    if whole:
        scales[page, :, :, block] = float("nan")


def _case(gpu, b, t, h, kv, d, page, starts, nodes, dtype):
    g = _gen(gpu, b, t, h, d)
    width = -(-(max(starts) + nodes) // page)
    codes, scales = _cache(gpu, g, b * width, kv, page, d, dtype)
    table = torch.randperm(b * width, device=gpu, generator=g).view(b, width).int()
    q = torch.randn(b, t, h, d, device=gpu, generator=g).bfloat16()
    return q, codes, scales, table


def _compare(gpu, q, codes, scales, table, starts, sets, new, nodes, unseen):
    args = (table, _i32(starts, gpu), sets.to(gpu), _i32(new, gpu))
    host = table.tolist()
    size = codes.shape[3] * BLOCK
    for n, block, first, whole in unseen:  # zeros there first
        page, part = host[n][block * BLOCK // size], block * BLOCK % size // BLOCK
        d = codes.shape[-1] // BLOCK
        raw = codes.view(torch.uint8)
        raw[page, 0, :, part].view(-1, d // 16, BLOCK, 16)[:, :, first:] = 0
        raw[page, 1, :, part].view(-1, d, BLOCK)[..., first:] = 0
    clean = kvc.tree_attention(q, codes, scales, *args, nodes=nodes)
    want = _exact(q, codes, scales, table, starts, sets, new, nodes)
    rows, off = want.norm(dim=-1), (clean.double() - want).norm(dim=-1)
    assert not clean[rows == 0].any()
    assert (off <= 4 * TWO_ROUNDINGS * rows).all() and off.norm() <= TWO_ROUNDINGS * rows.norm()
    for n, block, first, whole in unseen:
        _spoil(codes, scales, host[n][block * BLOCK // size], block * BLOCK % size // BLOCK, first, whole)
    assert torch.equal(kvc.tree_attention(q, codes, scales, *args, nodes=nodes), clean)


# batch, rows, heads, kv heads, d, page, starts, new, whether the batch's tiles are dealt
_RAGGED = [
    (2, 5, 2, 2, 64, 32, [28, 30], [5, 1], False), (2, 20, 4, 2, 128, 64, [40, 20], [20, 3], False),
    (3, 40, 2, 2, 64, 32, [3000, 20, 31], [2, 40, 1], False), (4, 64, 2, 1, 64, 64, [0, 1, 700, 64], [64, 1, 7, 0], None),
    (8, 25, 64, 8, 128, 64, [4000, 2000, 31, 60, 0, 700, 3999, 1], [25, 4, 1, 0, 25, 3, 2, 25], True),
    (8, 64, 64, 8, 64, 64, [30, 5000, 3000, 64, 4100, 5, 2047, 1], [3, 2, 64, 40, 33, 1, 1, 64], True),
    (70, 33, 8, 1, 64, 128, [100 + 7 * i for i in range(70)], [i % 34 for i in range(70)], None),
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new,dealt", _RAGGED)
def test_nodes_past_a_sequences_new_tokens_may_hold_anything(gpu, dtype, b, t, h, kv, d, page, starts, new, dealt):
    print(f"ragged trees: {dtype} b={b} t={t} h={h} kv={kv} d={d} starts={starts[:4]} new={new[:4]}", flush=True)
    q, codes, scales, table = _case(gpu, b, t, h, kv, d, page, starts, t, dtype)
    if dealt is not None:
        assert _dealt(gpu, b, t, h, kv, d, table.shape[1] * page) == dealt
    unseen = []
    for n, (start, count) in enumerate(zip(starts, new)):
        end, last = start + count, table.shape[1] * page // BLOCK
        if end % BLOCK and count:  # behind the last new token of its block, whose scale is a good one
            unseen.append((n, end // BLOCK, end % BLOCK, False))
        unseen += [(n, block, 0, True) for block in range(-(-end // BLOCK), last)]
    _compare(gpu, q, codes, scales, table, starts, _sets(torch.Generator().manual_seed(t), b, t), new, t, unseen)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,kv,rep,start", [(1, 1, 2, 1, 16), (1, 3, 2, 4, 1040), (2, 8, 2, 4, 16), (1, 40, 1, 2, 16),
                                             (8, 32, 8, 8, 4112), (8, 48, 8, 8, 5008)])
def test_a_block_of_nodes_that_no_row_sees_may_hold_anything(gpu, dtype, b, t, kv, rep, start):
    """Rows that see nodes of the first and of the last block: the one between them, the rest of the last one behind the
    last node that is seen, and the blocks after it."""
    d, page, nodes = 128, 32, 64
    starts = [start] * b
    q, codes, scales, table = _case(gpu, b, t, kv * rep, kv, d, page, [start + 64], nodes, dtype)
    assert _dealt(gpu, b, t, kv * rep, kv, d, table.shape[1] * page) == (b == 8)
    sets = torch.tensor([[1 << (i % 16) | (1 << 50 + i % 3 if i % 4 == 1 else 0) for i in range(t)]]).expand(b, t)
    seen = 53 if t > 5 else 52 if t > 1 else 1  # behind the last node seen: 50 + i % 3 of rows 1, 5, 9
    first, end = start // BLOCK, start + seen
    unseen = []
    for n in range(b):
        unseen += [(n, block, 0, True) for block in range(first + 1, first + 4) if t == 1 or block != end // BLOCK]
        unseen.append((n, end // BLOCK, end % BLOCK, False))
    _compare(gpu, q, codes, scales, table, starts, sets, None, nodes, unseen)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,kv,rep,start", [(1, 3, 2, 4, 1040), (2, 8, 2, 4, 16), (8, 32, 8, 8, 4112)])
def test_nodes_that_no_row_sees_within_a_block_change_nothing(gpu, dtype, b, t, kv, rep, start):
    """The largest finite codes at such places, the block's scales being those of the nodes that are seen."""
    d, page, nodes = 128, 32, 64
    q, codes, scales, table = _case(gpu, b, t, kv * rep, kv, d, page, [start], nodes, dtype)
    assert _dealt(gpu, b, t, kv * rep, kv, d, table.shape[1] * page) == (b == 8)
    seen = list(range(0, 63, 3))  # every third node
    sets = torch.tensor([[sum(1 << n for n in seen if n <= seen[i % 21]) for i in range(t)]])
    sets[0, -1] = sum(1 << n for n in seen)
    sets = sets.expand(b, t)
    args = (table, _i32([start] * b, gpu), sets.to(gpu))
    clean = kvc.tree_attention(q, codes, scales, *args, nodes=nodes)
    want = _exact(q, codes, scales, table, [start] * b, sets, None, nodes)
    assert (clean.double() - want).norm() <= TWO_ROUNDINGS * want.norm()
    raw, largest = codes.view(torch.uint8), 0x7e if dtype is torch.float8_e4m3fn else 127
    for token in (start + n for n in range(nodes) if n not in seen):
        pages, cell = table[:, token // page].long(), token % BLOCK
        raw[:, 0, :, 0].view(-1, kv, d // 16, BLOCK, 16)[pages, :, :, cell] = largest
        raw[:, 1, :, 0].view(-1, kv, d, BLOCK)[pages, :, :, cell] = largest
    assert torch.equal(kvc.tree_attention(q, codes, scales, *args, nodes=nodes), clean)
