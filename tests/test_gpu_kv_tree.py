"""Drafted trees over the paged 8-bit cache: norms and positions on the way in, attention over ancestors, keeping the
accepted nodes.

Codes and scales are compared bit for bit with 32-bit restatements (the norm's factor from 64 bits, as it is defined).
Attention is compared with float64; its tolerance is that of the attention without a tree: 2^-7 of the result's norm.
"""

from __future__ import annotations

import math

import pytest
import torch
from test_gpu_kv_cache import BLOCK, FORMATS, TWO_ROUNDINGS, _cells, _check_append, _gen, _pool, _quantised, _tables

from flextensor_amd import kv_cache as kvc

pytestmark = pytest.mark.gpu


def _i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu) if values is not None else None


def _normed(x, weight, eps):
    factor = torch.rsqrt(x.cpu().double().pow(2).mean(-1, keepdim=True) + eps).float()
    return x.cpu().float() * factor * weight.cpu().float()


def _turned(x, at, cos, sin):
    """fp32 rows [b, t, heads, d] turned by rows `at` of the tables; 0 where there is no such row."""
    ok = (at >= 0) & (at < cos.shape[0])
    c, s = (v.cpu()[at.clamp(0, cos.shape[0] - 1)].unsqueeze(2) for v in (cos, sin))
    d = x.shape[-1]
    y = x * c + torch.cat((-x[..., d // 2:], x[..., : d // 2]), -1) * s
    return torch.where(ok[..., None, None], y, 0.0), ok


# batch, tokens, heads, kv heads, d, page, starts, new
_APPEND = [
    (1, 1, 1, 1, 64, 32, [0], None), (1, 1, 4, 4, 128, 32, [31], None), (2, 7, 4, 4, 128, 64, [30, 57], [7, 3]),
    (3, 13, 6, 2, 64, 128, [5, 0, 200], [1, 0, 13]), (1, 64, 8, 2, 128, 64, [31], None),
    (1, 1060, 62, 62, 64, 64, [17], None), (2, 5, 2, 2, 64, 32, [-1, 93], None), (2, 33, 3, 1, 128, 32, [0, 60], None),
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("norm,tree", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new", _APPEND)
def test_append_with_norms_and_positions_is_the_definition(gpu, dtype, norm, tree, b, t, h, kv, d, page, starts, new):
    width = (max(starts) + t + page - 1) // page
    codes, scales = _pool(gpu, b * width + 2, kv, page, d, dtype)
    g = _gen(gpu, b, t, h, d)
    table = torch.randperm(codes.shape[0], device=gpu, generator=g)[: b * width].view(b, width).int()
    q = torch.randn(b, t, h, d, device=gpu, generator=g).mul(2.0).bfloat16()
    k, v = (torch.randn(b, t, kv, d, device=gpu, generator=g).mul(3.0 - 2.9 * i).bfloat16() for i in range(2))
    weights = [(1 + 0.3 * torch.randn(d, device=gpu, generator=g)).bfloat16() for _ in range(2)] if norm else [None] * 2
    cos, sin = _tables(d, width * page, gpu)
    at = torch.tensor(starts)[:, None] + torch.arange(t)
    if tree:
        at = torch.tensor(starts)[:, None].clamp(min=0) + torch.randint(0, 5, (b, t), generator=torch.Generator().manual_seed(1))
    old = codes.clone(), scales.clone()
    got = kvc.append(q, k, v, cos, sin, codes, scales, table, _i32(starts, gpu), _i32(new, gpu),
                     positions=_i32(at.tolist(), gpu) if tree else None, q_norm=weights[0], k_norm=weights[1], eps=1e-5)
    ready = [_normed(x, w, 1e-5) if norm else x.cpu().float() for x, w in zip((q, k), weights)]
    ready = [_turned(x, at, cos, sin)[0] for x in ready]
    still = torch.ones(width * page + t, d), torch.zeros(width * page + t, d)  # they have been turned
    _check_append(ready[0], ready[1], v, *still, old, codes, scales, table.cpu(), starts, new, got)


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_of_odd_norms_and_positions(gpu, dtype):
    """Rows of zeros, tiny and huge numbers, an infinity and a NaN; positions outside the tables; strided inputs."""
    b, t, h, kv, d, page = 2, 12, 4, 2, 128, 32
    g = _gen(gpu, 5)
    fused = torch.randn(b, t, h + 2 * kv, d, device=gpu, generator=g).bfloat16()
    q, k, v = fused[:, :, :h], fused[:, :, h: h + kv], fused[:, :, h + kv:]
    k[0, 1], k[0, 2], k[0, 3] = 0.0, 1e-30, 1e38
    q[0, 1], q[0, 2], q[0, 3] = 0.0, 1e-30, 1e38
    weights = [(1 + 0.3 * torch.randn(d, device=gpu, generator=g)).bfloat16() for _ in range(2)]
    codes, scales = _pool(gpu, 4, kv, page, d, dtype)
    table = _i32([[1, 3], [0, 2]], gpu)
    cos, sin = _tables(d, 40, gpu)
    at = torch.tensor([[7, 8, 8, 9, -1, 40, 39, 0, 1, 2, 3, 1 << 30], [20 + i // 3 for i in range(t)]])
    at_held = torch.zeros(b, t + 5, dtype=torch.int32, device=gpu)
    at_held[:, :t] = at.to(gpu)
    old = codes.clone(), scales.clone()
    got = kvc.append(q, k, v, cos, sin, codes, scales, table, _i32([5, 30], gpu), positions=at_held[:, :t],
                     q_norm=weights[0], k_norm=weights[1], eps=1e-6)
    (qr, ok), (kr, _) = (_turned(_normed(x, w, 1e-6), at, cos, sin) for x, w in zip((q, k), weights))
    vr = torch.where(ok[..., None, None], v.cpu().float(), 0.0)
    still = torch.ones(80, d), torch.zeros(80, d)
    _check_append(qr, kr, vr, *still, old, codes, scales, table.cpu(), [5, 30], None, got)
    k[0, 0, 0, 3], q[0, 0, 1, 5] = float("nan"), float("inf")
    got = kvc.append(q, k, v, cos, sin, codes, scales, table, _i32([5, 30], gpu), positions=at_held[:, :t],
                     q_norm=weights[0], k_norm=weights[1], eps=1e-6)
    assert got[0, 0, 1].isnan().any() and got[0, 0, 0].isfinite().all() and got[0, 1:].isfinite().all()


def _sets(g, b, t):
    """Random trees as sets of ancestors, the node's own bit included."""
    sets = torch.zeros(b, t, dtype=torch.int64)
    for n in range(b):
        for i in range(t):
            parent = int(torch.randint(-1, max(i, 1), (), generator=g)) if i else -1
            bit = (1 << i) - ((1 << 64) if i == 63 else 0)
            sets[n, i] = bit | (int(sets[n, parent]) if 0 <= parent < i else 0)
    return sets


def _tree64(q, codes, scales, table, starts, sets, new, nodes):
    b, t, h, d = q.shape
    kv, size, pages = codes.shape[2], codes.shape[3] * BLOCK, codes.shape[0]
    out = torch.zeros(b, t, h, d, dtype=torch.float64)
    q, scales, table = q.cpu().double(), scales.cpu().double(), table.cpu()
    cells = codes.cpu().float().double() * scales[..., None]
    keys = cells[:, 0].unflatten(-1, (d // 16, BLOCK, 16)).transpose(-3, -2).flatten(-2)  # [pages, kv, parts, 32, d]
    vals = cells[:, 1].unflatten(-1, (d, BLOCK)).transpose(-2, -1)
    for n in range(b):
        start = starts[n]
        if start < 0 or start > table.shape[1] * size:
            continue
        for i in range(max(0, min(new[n] if new is not None else t, t))):
            pos = torch.tensor([p for p in range(min(start + nodes, table.shape[1] * size))
                                if p < start or int(sets[n, i]) >> (p - start) & 1], dtype=torch.int64)
            page = table[n].long()[pos // size]
            ok = (page >= 0) & (page < pages)
            pos, page = pos[ok], page[ok]
            if not len(pos):
                continue
            part, cell = pos % size // BLOCK, pos % BLOCK
            for head in range(h):
                j = head // (h // kv)
                s = keys[page, j, part, cell] @ q[n, i, head] / math.sqrt(d)
                w = torch.exp(s - s.max())
                out[n, i, head] = (w / w.sum()) @ vals[page, j, part, cell]
    return out


# batch, rows, heads, kv heads, d, page, starts, new, nodes (None: the rows)
_TREES = [
    (1, 1, 1, 1, 64, 32, [0], None, None), (1, 2, 4, 4, 128, 64, [31], None, None), (1, 13, 4, 4, 128, 32, [100], None, None),
    (2, 5, 8, 2, 128, 64, [60, 0], [5, 2], None), (1, 64, 2, 1, 64, 64, [0], None, None), (1, 64, 8, 8, 128, 64, [33], None, 64),
    (2, 25, 16, 2, 128, 64, [300, 17], None, None), (3, 9, 6, 2, 64, 32, [5, -1, 90], [9, 9, 0], None),
    (2, 40, 8, 1, 128, 128, [1023, 1024], None, None), (1, 7, 4, 1, 64, 64, [5001], None, 40),   # a level of the nodes
    (1, 33, 6, 2, 128, 64, [2111], None, 50), (4, 3, 2, 2, 64, 32, [0, 0, 91, 400], [0, 3, 2, 3], 61),
    (1, 30, 4, 2, 64, 32, [70], None, 30),  # nodes that the table does not hold
    (2, 4, 2, 1, 64, 32, [96, 97], None, 0),  # a prefix that ends with the table, and one past it
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new,nodes", _TREES)
def test_tree_attention_matches_float64(gpu, dtype, b, t, h, kv, d, page, starts, new, nodes):
    print(f"tree: {dtype} b={b} t={t} h={h} kv={kv} d={d} page={page} starts={starts} new={new} nodes={nodes}", flush=True)
    held = t if nodes is None else nodes
    width = 3 if starts in ([70], [96, 97]) else (max(starts) + held + page - 1) // page
    codes, scales = _pool(gpu, b * width + 1, kv, page, d, dtype, seed=t)
    g = _gen(gpu, b, t, h, d, page)
    table = torch.randperm(codes.shape[0], device=gpu, generator=g)[: b * width].view(b, width).int()
    q = torch.randn(b, t, h, d, device=gpu, generator=g).mul(2.0).bfloat16()
    sets = _sets(torch.Generator().manual_seed(b + t), b, max(held, t))[:, -t:]  # the last ones, where rows are a level
    want = _tree64(q, codes, scales, table, starts, sets, new, held)
    for most in (None, max(starts) + held):
        got = kvc.tree_attention(q, codes, scales, table, _i32(starts, gpu), sets.to(gpu), _i32(new, gpu), nodes=nodes,
                                 max_tokens=most).cpu()
        assert (got.double() - want).norm() <= TWO_ROUNDINGS * want.norm()
        zero = ~want.flatten(2).any(-1)
        assert not got.flatten(2)[zero].any()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("t,h", [(5, 2), (40, 4)])
def test_a_chain_is_the_attention_without_a_tree(gpu, dtype, t, h):
    codes, scales = _pool(gpu, 20, 2, 64, 128, dtype)
    g = _gen(gpu, 9)
    table = torch.randperm(20, device=gpu, generator=g)[:18].view(2, 9).int()
    q = torch.randn(2, t, h, 128, device=gpu, generator=g).bfloat16()
    starts = _i32([300, 45], gpu)
    chain = torch.tensor([(2 << i) - 1 for i in range(t)], device=gpu).expand(2, t)
    got = kvc.tree_attention(q, codes, scales, table, starts, chain).double()
    want = kvc.attention(q, codes, scales, table, starts).double()
    # each is within the tolerance of the result in 64 bits, so within twice of each other: blocks that only one of them
    # masks round their scores once more
    assert (got - want).norm() <= 2 * TWO_ROUNDINGS * want.norm()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("t,rep", [(6, 1), (30, 4)])
def test_what_no_row_sees_has_no_part(gpu, dtype, t, rep):
    """Holes in the prefix, and what lies in the last block behind the nodes and in rows' own places that they do not
    see: the largest codes there change nothing; behind the nodes not even NaN codes do."""
    kv, d, page = 2, 64, 32
    codes, scales = _pool(gpu, 8, kv, page, d, dtype)
    table = _i32([[4, -1, 2, 9, 0, 6]], gpu)  # two holes
    g = _gen(gpu, t)
    q = torch.randn(1, t, kv * rep, d, device=gpu, generator=g).bfloat16()
    starts = 100 + 50
    sets = _sets(torch.Generator().manual_seed(t), 1, t)
    want = _tree64(q, codes, scales, table, [starts], sets, None, t)
    call = lambda: kvc.tree_attention(q, codes, scales, table, _i32([starts], gpu), sets.to(gpu))  # noqa: E731
    got = call()
    assert (got.cpu().double() - want).norm() <= TWO_ROUNDINGS * want.norm()
    raw = codes.view(torch.uint8)
    for part in (6,):  # page of tokens 160 .. 191: the nodes end at 150 + t
        keys = raw[part, 0].view(kv, 1, d // 16, BLOCK, 16)
        vals = raw[part, 1].view(kv, 1, d, BLOCK)
        first = max(0, starts + t - 160)
        keys[:, :, :, first:], vals[..., first:] = 127, 127
    assert torch.equal(call(), got)
    empty = torch.zeros_like(sets)
    assert not kvc.tree_attention(q, codes, scales, table, _i32([0], gpu), empty.to(gpu)).any()
    assert not kvc.tree_attention(q, codes, scales, _i32([[-1] * 6], gpu), _i32([starts], gpu), sets.to(gpu)).any()


def _check_keep(old, codes, scales, table, starts, path, counts):
    """Block by block on the CPU in 32 bits."""
    dtype = codes.dtype
    old_codes, old_scales, codes, scales = old[0].cpu(), old[1].cpu(), codes.cpu(), scales.cpu()
    layers, pages, _, kv, parts, bytes_ = codes.shape
    d, size = bytes_ // BLOCK, parts * BLOCK
    touched = torch.zeros(scales.shape, dtype=torch.bool)
    for n, start in enumerate(starts):
        places = []
        capacity = table.shape[1] * size
        for i in range(min(counts[n] if counts is not None else len(path[n]), len(path[n]))):
            p = path[n][i]
            if start < 0 or start + i >= capacity or p < i or p > 63 or start + p >= capacity or (i and p <= path[n][i - 1]):
                break
            places.append(start + p)
        if start < 0 or not places:
            continue
        for block in range(start // BLOCK, (start + len(places) - 1) // BLOCK + 1):
            page, part = int(table[n][block * BLOCK // size]), block % parts
            if not 0 <= page < pages:
                continue
            tokens = [p if p < start else places[p - start] for p in range(block * BLOCK, min((block + 1) * BLOCK, start + len(places)))]
            for layer in range(layers):
                for head in range(kv):
                    for side in range(2):
                        rows, was = [], []
                        for p in tokens:
                            at = int(table[n][p // size])
                            ok = 0 <= at < pages
                            rows.append(_cells(old_codes[layer], at, side, head, p // BLOCK % parts, d)[p % BLOCK] if ok
                                        else torch.zeros(d))
                            was.append(old_scales[layer, at, side, head, p // BLOCK % parts] if ok else torch.tensor(0.0))
                        was = torch.stack(was)
                        now = was.max()
                        inverse = 1.0 / now if now > 0 else torch.tensor(0.0)
                        ratio = torch.where(now > was, was * inverse, 1.0)[:, None]
                        want = torch.zeros(BLOCK, d)
                        want[: len(tokens)] = _quantised(torch.stack(rows) * ratio, dtype)
                        assert torch.equal(_cells(codes[layer], page, side, head, part, d).nan_to_num(999.0),
                                           want.nan_to_num(999.0)), (n, block, layer, head, side)
                        assert scales[layer, page, side, head, part] == now
                        touched[layer, page, side, head, part] = True
    same = ~touched
    assert torch.equal(codes.view(torch.uint8)[same], old_codes.view(torch.uint8)[same])
    assert torch.equal(scales[same], old_scales[same])


# kv heads, d, page, starts, path, counts
_KEEP = [
    (1, 64, 32, [0], [[0]], None), (2, 128, 64, [31], [[0, 1, 2]], None), (2, 128, 64, [30], [[0, 5, 40, 63]], None),
    (1, 128, 32, [10, 33], [[0, 3, 9, 20], [1, 2, 3, 4]], [4, 2]), (3, 64, 128, [100, 0, 7], [[2, 40]] * 3, [2, 0, 1]),
    (1, 64, 32, [5], [list(range(64))], None), (1, 128, 64, [31], [list(range(64))], None),
    (1, 64, 32, [0, 0, 0], [[0, 2, 2, 3], [3, 1, 5, 6], [0, 64, 65, 66]], None),  # paths that end early
    (1, 64, 32, [-1, 90, 96], [[0, 1, 2], [0, 4, 8], [0, 1, 2]], [3, 3, 3]),       # no part, the table's end, past it
    (1, 64, 32, [60], [[0, 1, 2, 3, 40]], [9]),
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("kv,d,page,starts,path,counts", _KEEP)
def test_keep_is_the_definition(gpu, dtype, kv, d, page, starts, path, counts):
    layers, b = 2, len(starts)
    width = 3 if 96 in starts else (max(starts) + 64 + page - 1) // page
    pools = [_pool(gpu, b * width + 2, kv, page, d, dtype, seed=i) for i in range(layers)]
    codes = torch.stack([p[0].view(torch.uint8) for p in pools]).view(dtype)
    scales = torch.stack([p[1] for p in pools])
    scales[1, :, 1] = 0.0  # blocks of zeros
    scales[0, :, 0, 0] = 0.25  # blocks of one scale: their codes move as they are
    table = torch.randperm(b * width + 2, device=gpu, generator=_gen(gpu, kv, d, page))[: b * width].view(b, width).int()
    if b > 2:
        table[2, -1] = -1
    old = codes.clone(), scales.clone()
    kvc.keep(codes, scales, table, _i32(starts, gpu), _i32(path, gpu), _i32(counts, gpu))
    _check_keep(old, codes, scales, table.cpu().tolist() and table.cpu(), starts, path, counts)


def test_refusals(gpu):
    codes, scales = _pool(gpu, 4, 2, 32, 64, torch.int8)
    table, starts = _i32([[0, 1]], gpu), _i32([3], gpu)
    q = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16, device=gpu)
    k = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16, device=gpu)
    cos, sin = _tables(64, 64, gpu)
    tree = torch.ones(1, 4, dtype=torch.int64, device=gpu)
    w = torch.ones(64, dtype=torch.bfloat16, device=gpu)

    def append(**more):
        return kvc.append(q, k, k, cos, sin, codes, scales, table, starts, **more)

    def attend(tree=tree, **more):
        return kvc.tree_attention(q, codes, scales, table, starts, tree, **more)

    def keep(path, counts=None, codes=codes[None], scales=scales[None]):
        return kvc.keep(codes, scales, table, starts, path, counts)

    for bad in (lambda: append(q_norm=w), lambda: append(k_norm=w), lambda: append(q_norm=w, k_norm=w[:32]),
                lambda: append(q_norm=w, k_norm=w, eps=-1.0), lambda: append(q_norm=w, k_norm=w, eps=float("nan")),
                lambda: append(positions=_i32([[1, 2, 3]], gpu)), lambda: append(positions=_i32([1, 2, 3, 4], gpu)),
                lambda: append(q_norm=w, k_norm=w.clone().requires_grad_()),
                lambda: append(positions=_i32([[1, 2, 3, 4]], gpu).cpu()),
                lambda: attend(tree[:, :3]), lambda: attend(tree[0]), lambda: attend(tree.cpu()),
                lambda: attend(nodes=65), lambda: attend(nodes=-1), lambda: attend(max_tokens=-1),
                lambda: attend(torch.ones(1, 8, dtype=torch.int64, device=gpu)[:, ::2]),
                lambda: keep(_i32([0, 1], gpu)), lambda: keep(_i32([list(range(65))], gpu)), lambda: keep(_i32([[0], [1]], gpu)),
                lambda: keep(_i32([[0]], gpu), _i32([1, 1], gpu)), lambda: keep(_i32([[0]], gpu), codes=codes, scales=scales),
                lambda: keep(_i32([[0]], gpu).cpu())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: append(q_norm=w.float(), k_norm=w), lambda: append(positions=torch.zeros(1, 4, device=gpu).long()),
                lambda: attend(tree.int()), lambda: keep(torch.zeros(1, 2, dtype=torch.int64, device=gpu))):
        with pytest.raises(TypeError):
            bad()
    assert kvc.tree_attention(q[:0], codes, scales, table[:0], starts[:0], tree[:0]).shape == (0, 4, 4, 64)
    keep(_i32([[]], gpu).int())
    kvc.keep(codes[None][:0], scales[None][:0], table, starts, _i32([[0]], gpu))
