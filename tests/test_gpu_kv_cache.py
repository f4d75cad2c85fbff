"""The paged 8-bit KV cache: writing, attention and page copies against plain restatements.

Codes and scales are compared bit for bit: the cache is defined by 32-bit operations that torch's elementary ones
make as well. Attention is compared with float64 over the numbers that the codes stand for; its tolerance is that of
the attention over a bf16 cache, an output rounded once from products whose probabilities were rounded: 2^-7.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from flextensor_amd import kv_cache as kvc

pytestmark = pytest.mark.gpu

BLOCK = 32
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FORMATS = list(TOP)
TWO_ROUNDINGS = 2.0 ** -7
ONE_ROUNDING = 2.0 ** -8


def _gen(gpu, *key: int) -> torch.Generator:
    return torch.Generator(device=gpu).manual_seed(sum(7 ** i * k for i, k in enumerate(key)) % 2 ** 31)


def _tables(d: int, n: int, gpu) -> tuple[torch.Tensor, torch.Tensor]:
    ang = torch.outer(torch.arange(n, dtype=torch.float32), 1.0 / 10000.0 ** (torch.arange(0, d, 2) / d))
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(gpu), ang.sin().to(gpu)


def _pool(gpu, pages: int, kv: int, page: int, d: int, dtype, seed: int = 0):
    g = _gen(gpu, pages, kv, page, d, seed)
    top = TOP[dtype]
    y = torch.randn(pages, 2, kv, page // BLOCK, BLOCK * d, device=gpu, generator=g).mul_(top / 4).clamp_(-top, top)
    codes = (y.round() if dtype == torch.int8 else y).to(dtype)
    scales = torch.exp(0.3 * torch.randn(codes.shape[:-1], device=gpu, generator=g)) * (4 / top)
    return codes, scales


def _quantised(y: torch.Tensor, dtype) -> torch.Tensor:
    """[...] fp32 values over their scale as codes' numbers."""
    y = y.clamp(-TOP[dtype], TOP[dtype])
    return (torch.nan_to_num(y).round().to(dtype) if dtype == torch.int8 else y.to(dtype)).float()


def _cells(codes: torch.Tensor, page: int, side: int, head: int, part: int, d: int) -> torch.Tensor:
    """One block's codes as numbers, [32, d]."""
    c = codes.view(torch.uint8)[page, side, head, part].view(codes.dtype).float()
    return c.view(d // 16, BLOCK, 16).transpose(0, 1).reshape(BLOCK, d) if side == 0 else c.view(d, BLOCK).t()


def _check_append(q, k, v, cos, sin, old, codes, scales, table, starts, new, got_q):
    """Token by token on the CPU in 32 bits, block by block."""
    dtype = codes.dtype
    old_codes, old_scales = old[0].cpu(), old[1].cpu()
    codes, scales = codes.cpu(), scales.cpu()
    q, k, v, cos, sin, got_q = (x.cpu() for x in (q, k, v, cos, sin, got_q))
    b, t, kv, d = k.shape
    size = codes.shape[3] * BLOCK
    touched = torch.zeros(scales.shape, dtype=torch.bool)

    def turn(x, pos):  # [tokens, heads, d]
        c, s = cos[pos].unsqueeze(1), sin[pos].unsqueeze(1)
        return x * c + torch.cat((-x[..., d // 2:], x[..., : d // 2]), -1) * s

    for n in range(b):
        start, count = int(starts[n]), min(t, int(new[n]) if new is not None else t)
        capacity = table.shape[1] * size
        count = max(0, min(count, capacity - start, cos.shape[0] - start)) if start >= 0 else 0
        pos = slice(start, start + count)
        assert torch.equal(got_q[n, :count], turn(q[n, :count].float(), pos).bfloat16()), n
        assert not got_q[n, count:].any(), n
        turned = turn(k[n, :count].float(), pos)
        for block in range(start // BLOCK, (start + count - 1) // BLOCK + 1) if count else ():
            page, part = int(table[n, block * BLOCK // size]), block % (size // BLOCK)
            if not 0 <= page < codes.shape[0]:
                continue
            lo, hi = max(start, block * BLOCK), min(start + count, block * BLOCK + BLOCK)
            before = lo - block * BLOCK
            for head in range(kv):
                for side in range(2):
                    y = (turned if side == 0 else v[n].float())[lo - start: hi - start, head]
                    was = old_scales[page, side, head, part] if before else torch.tensor(0.0)
                    made = torch.where(y.isfinite(), y.abs(), torch.tensor(0.0)).max() * torch.tensor(1 / TOP[dtype])
                    s = torch.maximum(was, torch.where(made < 2.0 ** -100, 0.0, made))
                    inverse = 1.0 / s if s > 0 else torch.tensor(0.0)
                    want = torch.zeros(BLOCK, d)
                    kept = _cells(old_codes, page, side, head, part, d)[:before]
                    want[:before] = _quantised(kept * (was * inverse), dtype) if s > was else kept
                    want[before: before + hi - lo] = _quantised(y * inverse, dtype)
                    got = _cells(codes, page, side, head, part, d)
                    assert torch.equal(got.nan_to_num(999.0), want.nan_to_num(999.0)), (n, block, head, side)
                    assert torch.equal(scales[page, side, head, part], s), (n, block, head, side)
                    touched[page, side, head, part] = True
    same = ~touched
    assert torch.equal(codes.view(torch.uint8)[same], old_codes.view(torch.uint8)[same])
    assert torch.equal(scales[same], old_scales[same])


# batch, tokens, heads, kv heads, d, page, starts, new (None: every token)
_APPEND = [
    (1, 1, 1, 1, 64, 32, [0], None), (1, 1, 4, 4, 128, 32, [31], None), (2, 1, 8, 2, 128, 64, [32, 63], None),
    (3, 1, 6, 2, 64, 128, [5, 0, 200], [1, 0, 1]), (2, 7, 4, 4, 128, 64, [30, 57], [7, 3]),
    (1, 33, 2, 1, 128, 32, [0], None), (1, 64, 2, 2, 64, 64, [31], None), (2, 97, 4, 2, 128, 64, [1, 64], [97, 50]),
    (1, 1060, 62, 62, 64, 64, [17], None),  # several heads a workgroup, not a whole number of them
    (2, 5, 2, 2, 64, 32, [-1, 93], None),  # a sequence that takes no part, one that ends at its table's end
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new", _APPEND)
def test_append_is_the_definition(gpu, dtype, b, t, h, kv, d, page, starts, new):
    """Codes, scales and rotated queries, bit for bit; every other block keeps its bits."""
    width = 3 if max(starts) < 3 * page - t else (max(starts) + t + page - 1) // page
    codes, scales = _pool(gpu, b * width + 2, kv, page, d, dtype)
    g = _gen(gpu, b, t, h, d)
    table = torch.randperm(codes.shape[0], device=gpu, generator=g)[: b * width].view(b, width).int()
    q = torch.randn(b, t, h, d, device=gpu, generator=g).bfloat16()
    k, v = (torch.randn(b, t, kv, d, device=gpu, generator=g).mul(3.0 - 2.9 * i).bfloat16() for i in range(2))
    cos, sin = _tables(d, width * page, gpu)
    old = codes.clone(), scales.clone()
    starts_t = torch.tensor(starts, dtype=torch.int32, device=gpu)
    new_t = torch.tensor(new, dtype=torch.int32, device=gpu) if new is not None else None
    got = kvc.append(q, k, v, cos, sin, codes, scales, table, starts_t, new_t)
    _check_append(q, k, v, cos, sin, old, codes, scales, table.cpu(), starts, new, got)


@pytest.mark.parametrize("dtype", FORMATS)
def test_append_of_strided_and_extreme_values(gpu, dtype):
    """Slices of a fused projection; zeros, infinities, NaN, the smallest and the largest numbers; a hole and a
    short rotary table are left out."""
    b, t, h, kv, d, page = 2, 40, 4, 2, 64, 32
    g = _gen(gpu, 3)
    fused = torch.randn(b, t, h + 2 * kv, d, device=gpu, generator=g).bfloat16()
    q, k, v = fused[:, :, :h], fused[:, :, h: h + kv], fused[:, :, h + kv:]
    v[0, 3, 0, 5], v[0, 3, 0, 6], v[0, 4, 1, 7] = float("inf"), float("-inf"), float("nan")
    v[0, 32:, 0] = 0.0                                   # a block of zeros
    v[1, :, 1] = 1e-36                                   # below the smallest scale
    v[1, :, 0] = torch.finfo(torch.bfloat16).max
    v[1, 3, 0] = 1.0
    codes, scales = _pool(gpu, 8, kv, page, d, dtype)
    table = torch.tensor([[1, 7, -1], [5, 8, 2]], dtype=torch.int32, device=gpu)  # -1, and one past the pool: holes
    cos, sin = _tables(d, 69, gpu)                       # the second sequence's last token has no position
    old = codes.clone(), scales.clone()
    starts = torch.tensor([0, 30], dtype=torch.int32, device=gpu)
    got = kvc.append(q, k, v, cos, sin, codes, scales, table, starts)
    _check_append(q, k, v, cos, sin, old, codes, scales, table.cpu(), [0, 30], None, got)


def _attend64(q, codes, scales, table, starts, new):
    """Row by row over the tokens that it sees."""
    b, t, h, d = q.shape
    kv, size, pages = codes.shape[2], codes.shape[3] * BLOCK, codes.shape[0]
    out = torch.zeros(b, t, h, d, dtype=torch.float64)
    q, scales, table = q.cpu().double(), scales.cpu().double(), table.cpu()
    cells = torch.stack([codes.cpu().view(torch.uint8).view(codes.dtype).float().double()])[0] * scales[..., None]
    keys = cells[:, 0].unflatten(-1, (d // 16, BLOCK, 16)).transpose(-3, -2).flatten(-2)  # [pages, kv, parts, 32, d]
    vals = cells[:, 1].unflatten(-1, (d, BLOCK)).transpose(-2, -1)
    for n in range(b):
        start = starts[n]
        if start < 0:
            continue
        count = max(0, min(new[n] if new is not None else t, t, table.shape[1] * size - start))
        for i in range(count):
            pos = torch.arange(start + i + 1)
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


# batch, tokens, heads, kv heads, d, page, starts, new
_ATTEND = [
    (1, 1, 1, 1, 64, 32, [0], None), (1, 1, 4, 4, 128, 64, [31], None), (1, 1, 8, 1, 128, 32, [32], None),
    (2, 1, 16, 2, 128, 64, [300, 17], None), (3, 1, 6, 2, 64, 32, [5, -1, 700], [1, 1, 1]),
    (2, 1, 40, 2, 64, 128, [1023, 1024], None),                                       # more than one tile of rows
    (1, 1, 32, 32, 128, 64, [2100], None), (1, 1, 4, 1, 64, 64, [9001], None),        # split over the keys
    (2, 5, 8, 2, 128, 64, [60, 0], [5, 2]), (1, 17, 4, 4, 64, 32, [0], None), (1, 70, 6, 2, 128, 64, [45], None),
    (2, 130, 2, 1, 64, 32, [0, 333], [130, 77]), (1, 3, 12, 4, 128, 128, [4000], None),
    (4, 9, 2, 2, 64, 32, [0, 0, 91, 400], [0, 9, 5, 9]),
]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new", _ATTEND)
def test_attention_matches_float64(gpu, dtype, b, t, h, kv, d, page, starts, new):
    """Every tensor element past a sequence's last token is NaN (of the e4m3 codes) or has a NaN scale."""
    width = (max(starts) + t + page - 1) // page
    codes, scales = _pool(gpu, b * width + 1, kv, page, d, dtype)
    g = _gen(gpu, b, t, h, d, page)
    table = torch.randperm(codes.shape[0], device=gpu, generator=g)[: b * width].view(b, width).int()
    for n, start in enumerate(starts):
        end = start + (new[n] if new is not None else t)
        for block in range(max(0, end) // BLOCK, width * page // BLOCK):
            page_n, part, inside = int(table[n, block * BLOCK // page]), block % (page // BLOCK), max(0, end - block * BLOCK)
            if inside == 0:
                scales[page_n, :, :, part] = float("nan")
            if dtype != torch.int8:
                c = codes.view(torch.uint8)[page_n, :, :, part]
                c[0].view(kv, d // 16, BLOCK, 16)[:, :, inside:] = 0x7F
                c[1].view(kv, d, BLOCK)[..., inside:] = 0xFF
    q = torch.randn(b, t, h, d, device=gpu, generator=g).mul(2.0).bfloat16()
    starts_t = torch.tensor(starts, dtype=torch.int32, device=gpu)
    new_t = torch.tensor(new, dtype=torch.int32, device=gpu) if new is not None else None
    want = _attend64(q, codes, scales, table, starts, new)
    for longest in (None, max(starts) + t, 1):  # the caller's idea of the longest sequence changes no result
        got = kvc.attention(q, codes, scales, table, starts_t, new_t, max_tokens=longest).cpu().double()
        assert got.isfinite().all()
        assert (got - want).norm() <= TWO_ROUNDINGS * want.norm()
        rows = want.norm(dim=-1)
        assert ((got - want).norm(dim=-1) <= 4 * TWO_ROUNDINGS * rows.clamp(min=1e-30)).all()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("t,start", [(1, 250), (1, 4000), (20, 250), (200, 100)])
def test_attention_over_holes(gpu, dtype, t, start):
    """Pages that are not in the pool are not seen; a sequence of holes gives zeros."""
    kv, h, d, page = 2, 4, 128, 32
    width = (start + t + page - 1) // page
    codes, scales = _pool(gpu, 2 * width, kv, page, d, dtype)
    g = _gen(gpu, t, start)
    table = torch.randperm(2 * width, device=gpu, generator=g).view(2, width).int()
    table[0, ::3], table[0, 1::5] = -1, 2 * width
    table[1] = 1 << 30
    q = torch.randn(2, t, h, d, device=gpu, generator=g).bfloat16()
    starts = torch.tensor([start, start], dtype=torch.int32, device=gpu)
    want = _attend64(q, codes, scales, table, [start, start], None)
    got = kvc.attention(q, codes, scales, table, starts).cpu().double()
    assert (got - want).norm() <= TWO_ROUNDINGS * want.norm()
    assert not got[1].any()


def test_attention_of_extreme_scores(gpu):
    """Scores far apart, a block of a zero scale, and queries of another layout than the cache's heads."""
    kv, h, d, page, n = 2, 8, 64, 32, 500
    codes, scales = _pool(gpu, 17, kv, page, d, torch.int8)
    scales[3] = 0.0
    scales[5, 0] *= 300.0
    table = torch.arange(16, dtype=torch.int32, device=gpu).view(1, 16)
    g = _gen(gpu, 5)
    q = torch.randn(1, h, 3, d, device=gpu, generator=g).bfloat16().transpose(1, 2)
    starts = torch.tensor([n], dtype=torch.int32, device=gpu)
    want = _attend64(q, codes, scales, table, [n], None)
    got = kvc.attention(q, codes, scales, table, starts).cpu().double()
    assert (got - want).norm() <= TWO_ROUNDINGS * want.norm()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("layers,pages,kv,page,d,n", [(1, 2, 1, 32, 64, 1), (3, 9, 3, 64, 128, 4), (2, 700, 2, 32, 64, 300)])
def test_copy_pages_copies_bytes(gpu, dtype, layers, pages, kv, page, d, n):
    codes, scales = _pool(gpu, layers * pages, kv, page, d, dtype)
    codes, scales = codes.unflatten(0, (layers, pages)), scales.unflatten(0, (layers, pages))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n: 2 * n]
    want, want_scales = codes.view(torch.uint8).clone(), scales.clone()
    want[:, dst], want_scales[:, dst] = want[:, src], want_scales[:, src]
    kvc.copy_pages(codes, scales, src, dst)
    assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, want_scales)


def _attend64_gpu(q, codes, scales, table, starts, new):
    """The same on the GPU, head by head, for prompts."""
    b, t, h, d = q.shape
    kv, size = codes.shape[2], codes.shape[3] * BLOCK
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=q.device)
    for n in range(b):
        count = new[n] if new is not None else t
        length = starts[n] + count
        keys, vals = (x[0, :length].double() for x in kvc.read(codes, scales, table[n: n + 1, : -(-length // size)]))
        seen = torch.arange(length, device=q.device) <= starts[n] + torch.arange(count, device=q.device)[:, None]
        for head in range(h):
            j = head // (h // kv)
            s = (q[n, :count, head].double() @ keys[:, j].t().contiguous() / math.sqrt(d)).masked_fill(~seen, -math.inf)
            out[n, :count, head] = torch.softmax(s, -1) @ vals[:, j].contiguous()
    return out


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("b,t,h,kv,d,page,starts,new", [
    (1, 300, 64, 64, 128, 64, [0], None), (2, 290, 64, 64, 64, 32, [33, 0], [290, 1]),  # tiles of 256 rows, unsplit
    (1, 257, 128, 128, 128, 128, [511], None),
    (1, 64, 64, 8, 128, 64, [30000], None), (2, 300, 24, 8, 64, 64, [9000, 20], [300, 299]),  # and split over the keys
])
def test_prompts_match_float64(gpu, dtype, b, t, h, kv, d, page, starts, new):
    width = (max(starts) + t + page - 1) // page
    codes, scales = _pool(gpu, b * width, kv, page, d, dtype)
    g = _gen(gpu, b, t, h, d, page)
    table = torch.randperm(b * width, device=gpu, generator=g).view(b, width).int()
    q = torch.randn(b, t, h, d, device=gpu, generator=g).mul(2.0).bfloat16()
    starts_t = torch.tensor(starts, dtype=torch.int32, device=gpu)
    new_t = torch.tensor(new, dtype=torch.int32, device=gpu) if new is not None else None
    want = _attend64_gpu(q, codes, scales, table, starts, new)
    got = kvc.attention(q, codes, scales, table, starts_t, new_t).double()
    assert (got - want).norm() <= TWO_ROUNDINGS * want.norm()
    assert ((got - want).norm(dim=-1) <= 4 * TWO_ROUNDINGS * want.norm(dim=-1).clamp(min=1e-30)).all()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("t", [1, 40])
def test_both_host_paths_are_the_same_operations(gpu, dtype, t, monkeypatch):
    """The binding's calls and the Python functions behind them end in the same launches; both count as a write."""
    b, h, kv, d, page = 3, 4, 2, 64, 32
    results = []
    for plain in (False, True):
        if plain:
            nothing = lambda *args: None
            calls = SimpleNamespace(append=nothing, attention=nothing, copy_pages=nothing)
            monkeypatch.setattr(kvc.nat, "torch_calls", lambda: calls)
        codes, scales = _pool(gpu, 9, kv, page, d, dtype)
        table = torch.tensor([[0, 1, 2], [3, 4, 5], [6, 7, 8]], dtype=torch.int32, device=gpu)
        starts = torch.tensor([0, 31, -1], dtype=torch.int32, device=gpu)
        x = torch.randn(b, t, h + 2 * kv, d, device=gpu, generator=_gen(gpu, t)).to(torch.bfloat16)
        cos, sin = _tables(d, 96, gpu)
        versions = codes._version, scales._version
        q = kvc.append(x[:, :, :h], x[:, :, h:h + kv], x[:, :, h + kv:], cos, sin, codes, scales, table, starts)
        assert codes._version > versions[0] and scales._version > versions[1]
        y = kvc.attention(q, codes, scales, table, starts, max_tokens=80, scale=0.2)
        pool, pool_scales = codes[None].clone(), scales[None].clone()
        version = pool._version
        kvc.copy_pages(pool, pool_scales, [0, 3], [7, 8])
        assert pool._version > version
        results.append([r.view(torch.uint8) for r in (q, codes, scales, y, pool, pool_scales)])
    for one, other in zip(*results):
        assert torch.equal(one, other)


def test_forward_differentiation_is_refused(gpu):
    codes, scales = _pool(gpu, 1, 1, 32, 64, torch.int8)
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    q = torch.zeros(1, 1, 1, 64, device=gpu, dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises((TypeError, ValueError, RuntimeError, NotImplementedError)):
            kvc.attention(dual, codes, scales, table, table[:, 0])
