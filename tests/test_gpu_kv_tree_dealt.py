"""Attention of many trees, whose tiles of keys are dealt to the workgroups by the lengths that the device holds: heads
that many workgroups share, workgroups that have many heads, sequences without rows or keys among them.

The result is compared with float64 of the same codes; its tolerance is that of the attention without a tree, 2^-7 of
each row's norm: the probabilities and the result are rounded to bf16 once each.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from test_gpu_kv_cache import BLOCK, FORMATS, TWO_ROUNDINGS, _gen
from test_gpu_kv_tree import _i32, _sets

from flextensor_amd import _native as nat
from flextensor_amd import kv_cache as kvc

pytestmark = pytest.mark.gpu


def _cache(gpu, g, pages, kv, page, d, dtype):
    scales = torch.rand(pages, 2, kv, page // BLOCK, device=gpu, generator=g) * 0.02 + 0.001
    shape = (pages, 2, kv, page // BLOCK, BLOCK * d)
    if dtype is torch.int8:
        return torch.randint(-127, 128, shape, device=gpu, generator=g).to(dtype), scales
    return torch.randn(shape, device=gpu, generator=g).mul(20).to(dtype), scales


def _exact(q, codes, scales, table, starts, sets, new, nodes):
    """float64 [b, t, heads, d], a sequence at a time."""
    b, t, h, d = q.shape
    kv, size, pages = codes.shape[2], codes.shape[3] * BLOCK, codes.shape[0]
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=q.device)
    for n, start in enumerate(starts):
        count = max(0, min(t, new[n] if new is not None else t))
        held = min(start + nodes, table.shape[1] * size)
        if start < 0 or start > table.shape[1] * size or not count or not held:
            continue
        pos = torch.arange(held, device=q.device)
        page = table[n].long()[pos // size]
        ok = (page >= 0) & (page < pages)
        page = page.clamp(0, pages - 1)
        part, cell = pos % size // BLOCK, pos % BLOCK
        raw = codes.view(torch.uint8)  # tokens are picked before they are widened
        sides = (raw.unflatten(-1, (d // 16, BLOCK, 16))[page, 0, :, part, :, cell].flatten(2),
                 raw.unflatten(-1, (d, BLOCK))[page, 1, :, part, :, cell])  # [held, kv, d]
        keys, vals = (x.contiguous().view(codes.dtype).float().double() * scales.double()[page, i, :, part][..., None]
                      for i, x in enumerate(sides))
        bits = (sets[n, :count, None].to(q.device) >> (pos - start).clamp(0, 63)) & 1
        seen = ok & ((pos < start) | (bits == 1))  # [count, held]
        for j in range(kv):
            heads = slice(j * (h // kv), (j + 1) * (h // kv))
            s = (q[n, :count, heads].double().flatten(0, 1) @ keys[:, j].T.contiguous() / math.sqrt(d)).view(count, -1, held)
            s = s.masked_fill(~seen[:, None], float("-inf"))
            w = torch.exp(s - s.amax(-1, keepdim=True)).nan_to_num(0.0)
            total = w.sum(-1, keepdim=True)
            o = (w.flatten(0, 1) @ vals[:, j].contiguous()).view(count, -1, d)
            out[n, :count, heads] = torch.where(total > 0, o / total, 0.0)
    return out


def _dealt(gpu, b, t, h, kv, d, longest):
    """Whether such a call has the workspace of dealt tiles: two places of the rows, and a record, for each CU."""
    got = ctypes.c_size_t(0)
    nat.call("ftx_kv8_tree_attention_workspace", b, t, h, kv, d, longest, ctypes.byref(got))
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    return got.value == cus * (2 * min(t * h // kv, 256) * (d + 2) + 4) * 4


def _case(gpu, b, t, h, kv, d, page, longest, nodes, dtype, seed=0):
    """Ragged sequences, some of them without cached tokens, rows or a valid start, on pages with holes."""
    g = _gen(gpu, b, t, h, seed)
    host = torch.Generator().manual_seed(seed)
    width = -(-(longest + nodes) // page)
    pages = min(b * width, 600)  # sequences may share pages: nothing is written
    codes, scales = _cache(gpu, g, pages, kv, page, d, dtype)
    table = torch.randint(0, pages, (b, width), device=gpu, generator=g).int()
    starts = torch.randint(0, longest + 1, (b,), generator=host).tolist()
    new = torch.randint(0, t + 1, (b,), generator=host).tolist()
    starts[0], new[0] = longest, t
    if b > 4:
        starts[1], new[2], starts[3], starts[b - 1], new[b - 1] = 0, 0, -1, 0, 0
        table[4, 0] = -1
    q = torch.randn(b, t, h, d, device=gpu, generator=g).bfloat16()
    sets = _sets(host, b, min(t, 64))
    if t > 64:  # rows that share their sets
        sets = sets[:, torch.arange(t) % 64]
    return q, codes, scales, table, starts, sets, new


def _check(got, want):
    rows = want.norm(dim=-1)
    off = (got.double() - want).norm(dim=-1)
    assert not got[rows == 0].any()
    assert (off <= 4 * TWO_ROUNDINGS * rows).all() and off.norm() <= TWO_ROUNDINGS * rows.norm()


# batch, rows, heads, kv heads, d, page, longest, nodes
_CASES = [
    (130, 64, 16, 2, 128, 32, 300, 64),   # more sequences than a wave has lanes, many heads for a workgroup
    (67, 33, 16, 2, 64, 64, 900, 33),     # 264 rows: tiles of 32 rows serve them better
    (67, 64, 16, 2, 64, 64, 900, 64),
    (4, 16, 32, 4, 128, 64, 32000, 16),   # many workgroups for a head
    (9, 300, 8, 1, 128, 128, 3000, 64),   # more rows than nodes, tiles of rows without any
    (40, 31, 40, 8, 128, 64, 1500, 31),   # 155 rows
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,longest,nodes", _CASES)
def test_dealt_trees_are_the_softmax_of_what_they_see(gpu, dtype, b, t, h, kv, d, page, longest, nodes):
    assert _dealt(gpu, b, t, h, kv, d, longest + nodes) == (t * h // kv != 264)
    q, codes, scales, table, starts, sets, new = _case(gpu, b, t, h, kv, d, page, longest, nodes, dtype)
    got = kvc.tree_attention(q, codes, scales, table, _i32(starts, gpu), sets.to(gpu), _i32(new, gpu), nodes=nodes,
                             max_tokens=longest + nodes)
    _check(got, _exact(q, codes, scales, table, starts, sets, new, nodes))


@pytest.mark.parametrize("starts", [[0] * 130, [-1] * 130, [300] + [-1] * 129, [-1] * 129 + [300], [31] * 130])
def test_batches_with_little_or_nothing_to_deal(gpu, starts):
    """Nothing at all, one sequence at either end, and all the same; the output held NaNs before."""
    b, t, h, kv, d, page, longest, nodes = _CASES[0]
    q, codes, scales, table, _, sets, _ = _case(gpu, b, t, h, kv, d, page, longest, nodes, torch.int8)
    if starts[0] == 0:
        nodes = 0
    for x in (torch.empty_like(q) for _ in range(3)):  # memory that the result may get
        x.fill_(float("nan"))
        del x
    got = kvc.tree_attention(q, codes, scales, table, _i32(starts, gpu), sets.to(gpu), nodes=nodes, max_tokens=longest + 64)
    _check(got, _exact(q, codes, scales, table, starts, sets, None, nodes))


def test_rows_left_out_may_hold_anything(gpu):
    """NaNs and infinities in the queries of rows that are left out reach no other row, and their results are 0."""
    b, t, h, kv, d, page, longest, nodes = _CASES[0]
    q, codes, scales, table, starts, sets, new = _case(gpu, b, t, h, kv, d, page, longest, nodes, torch.float8_e4m3fn, 1)
    args = (codes, scales, table, _i32(starts, gpu), sets.to(gpu), _i32(new, gpu))
    want = _exact(q, codes, scales, table, starts, sets, new, nodes)
    out = torch.arange(t, device=gpu)[None] >= _i32(new, gpu)[:, None]
    q[out] = torch.tensor([float("nan"), float("inf")], device=gpu).bfloat16().repeat(d // 2)
    _check(kvc.tree_attention(q, *args, nodes=nodes, max_tokens=longest + nodes), want)


def test_a_captured_call_deals_by_the_lengths_of_each_replay(gpu):
    b, t, h, kv, d, page, longest, nodes = _CASES[2]
    q, codes, scales, table, starts, sets, new = _case(gpu, b, t, h, kv, d, page, longest, nodes, torch.int8)
    at, count, tree = _i32(starts, gpu), _i32(new, gpu), sets.to(gpu)

    def run():
        return kvc.tree_attention(q, codes, scales, table, at, tree, count, nodes=nodes, max_tokens=longest + nodes)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(5):
        host = torch.Generator().manual_seed(seed)
        at.copy_(torch.randint(-1 if seed else longest, longest + 1, (b,), generator=host))
        count.copy_(torch.randint(0 if seed else t, t + 1, (b,), generator=host))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want)


def test_more_tiles_of_keys_than_are_counted_are_refused(gpu):
    """Tiles are dealt in 32-bit numbers: 4096 tables of two million tokens hold too many. Nothing is launched."""
    b, t, h, kv, d = 4096, 64, 64, 8, 64
    codes, scales = _cache(gpu, _gen(gpu, 0), 1, kv, 64, d, torch.int8)
    table = torch.zeros(b, 1 << 15, dtype=torch.int32, device=gpu)
    starts = torch.zeros(b, dtype=torch.int32, device=gpu)
    q = torch.empty(b, t, h, d, dtype=torch.bfloat16, device=gpu)
    sets = torch.ones(1, t, dtype=torch.int64, device=gpu).expand(b, t)
    with pytest.raises(nat.FtxError, match="tiles of keys"):
        kvc.tree_attention(q, codes, scales, table, starts, sets, max_tokens=64)
