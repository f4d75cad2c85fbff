"""The paged cache's bookkeeping and layout, and what its operations and the int8 linear refuse, without a GPU."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from flextensor_amd import _native as nat
from flextensor_amd import hip, kv_cache as kvc
from flextensor_amd import workloads as W


@pytest.fixture
def pool(monkeypatch):
    """A small pool whose page copies are torch's, and a record of them."""
    copies = []

    def copy(codes, scales, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        copies.append((list(src), list(dst)))
        codes.view(torch.uint8)[:, dst] = codes.view(torch.uint8)[:, src]
        scales[:, dst] = scales[:, src]

    monkeypatch.setattr(kvc, "copy_pages", copy)
    cache = kvc.PagedKVCache(2, 1, 64, 8, page_tokens=32, dtype=torch.int8, device="cpu")
    for p in range(cache.pages):
        cache.codes[:, p], cache.scales[:, p] = p, float(p)
    cache.copies = copies
    return cache


def _write(cache, step, marks):
    """Marks the page of each sequence's first new token: what an append would write."""
    for s, mark in zip(step.sequences, marks):
        page = cache.table(s)[cache.length(s) // cache.page_tokens]
        cache.codes[:, page] = mark
    cache.commit(step)


def test_steps_reserve_pages_and_carry_the_tables(pool):
    a, b = pool.open(), pool.open()
    step = pool.begin([a, b], [40, 3])
    assert step.tokens == 40 and step.max_tokens == 40 and pool.free_pages == 5
    assert step.table.dtype == step.starts.dtype == step.new.dtype == torch.int32
    assert step.table.tolist() == [pool.table(a), [*pool.table(b), -1]]
    assert step.starts.tolist() == [0, 0] and step.new.tolist() == [40, 3]
    pool.commit(step)
    step = pool.begin([b, a], 1)
    assert step.starts.tolist() == [3, 40] and step.max_tokens == 41 and pool.free_pages == 5 and not pool.copies
    assert step.layer(1).index == 1 and step.layer(0).step is step
    assert pool.page_bytes == 2 * 2 * (32 * 64 + 4)


def test_a_full_pool_changes_nothing(pool):
    a, b = pool.open(), pool.open()
    pool.commit(pool.begin([a], [7 * 32]))
    before = pool.table(a), pool.free_pages
    with pytest.raises(kvc.KVCacheFull):
        pool.begin([a, b], [1, 33])
    assert (pool.table(a), pool.free_pages) == before and pool.table(b) == []
    pool.close(a)
    assert pool.free_pages == 8
    with pytest.raises(KeyError):
        pool.length(a)


def test_forks_share_pages_until_one_of_them_writes(pool):
    a = pool.open()
    pool.commit(pool.begin([a], 40))
    b, c = pool.fork(a), pool.fork(a)
    first, last = pool.table(a)
    assert pool.table(b) == pool.table(c) == [first, last] and pool.free_pages == 6
    step = pool.begin([a, b, c], 1)  # all three write into the shared last page: two copies, the last keeps it
    assert pool.free_pages == 4 and len(pool.copies) == 1 and pool.copies[0][0] == [last, last]
    assert {pool.table(s)[0] for s in (a, b, c)} == {first}
    assert len({pool.table(s)[1] for s in (a, b, c)}) == 3 and pool.table(c)[1] == last
    assert all((pool.codes[:, pool.table(s)[1]] == last).all() for s in (a, b, c))
    _write(pool, step, (101, 102, 103))
    assert [int(pool.codes[0, pool.table(s)[1]].flatten()[0]) for s in (a, b, c)] == [101, 102, 103]
    pool.close(b)
    assert pool.free_pages == 5  # the first page is still shared by two


def test_forks_at_a_page_boundary_copy_nothing(pool):
    a = pool.open()
    pool.commit(pool.begin([a], 32))
    b = pool.fork(a)
    pool.commit(pool.begin([a, b], 1))
    assert not pool.copies and pool.table(a)[0] == pool.table(b)[0] and pool.table(a)[1] != pool.table(b)[1]


def test_truncated_sequences_give_pages_back_and_copy_what_they_share(pool):
    a = pool.open()
    pool.commit(pool.begin([a], 70))
    b = pool.fork(a)
    pool.truncate(b, 33)
    assert pool.length(b) == 33 and len(pool.table(b)) == 2 and pool.free_pages == 5
    pool.truncate(b, 5)
    step = pool.begin([b], 2)  # into the page that a shares
    assert pool.copies == [([pool.table(a)[0]], [pool.table(b)[0]])]
    pool.commit(step)
    with pytest.raises(ValueError):
        pool.truncate(b, 8)
    pool.truncate(a, 0)
    assert pool.table(a) == [] and pool.free_pages == 7


def test_compaction_moves_the_fewest_pages_and_resize_keeps_them(pool):
    seqs = [pool.open() for _ in range(4)]
    for s in seqs:
        pool.commit(pool.begin([s], 50))
    for s in (seqs[0], seqs[2]):
        pool.close(s)
    shared = pool.fork(seqs[3])
    content = {s: [int(pool.codes[0, p].flatten()[0]) for p in pool.table(s)] for s in (seqs[1], seqs[3], shared)}
    assert pool.compact() == 2
    assert sorted({p for s in (seqs[1], seqs[3]) for p in pool.table(s)}) == [0, 1, 2, 3]
    assert pool.table(shared) == pool.table(seqs[3])
    assert {s: [int(pool.codes[0, p].flatten()[0]) for p in pool.table(s)] for s in content} == content
    with pytest.raises(ValueError):
        pool.resize(3)
    pool.resize(4)
    assert pool.pages == 4 and pool.free_pages == 0 and pool.compact() == 0
    assert {s: [int(pool.codes[0, p].flatten()[0]) for p in pool.table(s)] for s in content} == content
    pool.resize(9)
    assert pool.free_pages == 5
    step = pool.begin([seqs[1]], 40)
    assert pool.table(seqs[1])[2] == 4 and step.max_tokens == 90


def test_a_long_run_keeps_every_reference(pool):
    """Random forks, steps, truncations, closings and compactions: a page is free or counted as often as it is held."""
    rng = random.Random(5)
    held: list[int] = []
    for _ in range(600):
        move = rng.choice(["open", "step", "step", "fork", "truncate", "close", "compact"])
        try:
            if move == "open":
                held.append(pool.open())
            elif move == "compact":
                pool.compact()
            elif held:
                s = rng.choice(held)
                if move == "step":
                    some = rng.sample(held, rng.randint(1, len(held)))
                    pool.commit(pool.begin(some, [rng.randint(0, 40) for _ in some]))
                elif move == "fork":
                    held.append(pool.fork(s))
                elif move == "truncate":
                    pool.truncate(s, rng.randint(0, pool.length(s)))
                else:
                    pool.close(s)
                    held.remove(s)
        except kvc.KVCacheFull:
            pass
        counts = [0] * pool.pages
        for s in held:
            assert len(pool.table(s)) >= -(-pool.length(s) // 32)
            for p in pool.table(s):
                counts[p] += 1
        assert counts == pool._refs
        assert sorted(pool._free) == [p for p in range(pool.pages) if not counts[p]]


def test_steps_refuse_what_does_not_fit(pool):
    a = pool.open()
    for call in (lambda: pool.begin([a, a], 1), lambda: pool.begin([a], [1, 2]), lambda: pool.begin([a], [5], tokens=4),
                 lambda: pool.begin([a], [-1])):
        with pytest.raises(ValueError):
            call()
    for args in ((0, 1, 64, 4), (1, 1, 96, 4), (1, 1, 64, 0)):
        with pytest.raises(ValueError):
            kvc.PagedKVCache(*args, device="cpu")
    with pytest.raises(ValueError):
        kvc.PagedKVCache(1, 1, 64, 4, page_tokens=48, device="cpu")
    with pytest.raises(TypeError):
        kvc.PagedKVCache(1, 1, 64, 4, dtype=torch.uint8, device="cpu")


def test_read_turns_blocks_into_tokens():
    """Keys lie as [d / 16, 32, 16], values as [d, 32], block by block of a page."""
    d, kv, page = 64, 2, 64
    keys = torch.randint(-127, 128, (3, page, kv, d), dtype=torch.int8)
    vals = torch.randint(-127, 128, (3, page, kv, d), dtype=torch.int8)
    codes = torch.empty(3, 2, kv, 2, 32 * d, dtype=torch.int8)
    for p in range(3):
        for head in range(kv):
            for block in range(2):
                k, v = keys[p, 32 * block: 32 * block + 32, head], vals[p, 32 * block: 32 * block + 32, head]
                codes[p, 0, head, block] = k.view(32, d // 16, 16).transpose(0, 1).reshape(-1)
                codes[p, 1, head, block] = v.t().reshape(-1)
    scales = torch.arange(1.0, 25.0).view(3, 2, kv, 2)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    got_k, got_v = kvc.read(codes, scales, table)
    assert got_k.shape == (1, 128, kv, d)
    for i, p in enumerate((2, 0)):
        rows = slice(64 * i, 64 * i + 64)
        for side, (got, want) in enumerate(((got_k, keys), (got_v, vals))):
            s = scales[p, side].t().repeat_interleave(32, 0).unsqueeze(-1)  # [tokens, kv, 1]
            assert torch.equal(got[0, rows], want[p].float() * s)


def test_operations_refuse_tensors_of_the_host():
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 2, 1, 1, 2048, dtype=torch.int8), torch.zeros(4, 2, 1, 1)
    table, starts = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="current GPU"):
        kvc.attention(q, codes, scales, table, starts)
    with pytest.raises(ValueError, match="current GPU"):
        kvc.append(q, q[:, :, :1], q[:, :, :1], torch.zeros(8, 64), torch.zeros(8, 64), codes, scales, table, starts)
    with pytest.raises(ValueError, match="current GPU"):
        kvc.copy_pages(codes[None], scales[None], [0], [1])
    with pytest.raises(ValueError, match="current GPU"):
        hip.int8_quantize(q.view(2, 64))
    with pytest.raises(TypeError, match="bf16"):
        hip.int8_linear(torch.zeros(2, 64), torch.zeros(3, 64, dtype=torch.int8), torch.ones(3))


def test_the_c_entries_refuse_before_they_touch_a_device():
    lib, nul = nat.load(), None
    b = ctypes.c_size_t(7)
    work = lib.ftx_kv8_attention_workspace
    for shape, code in (((1, 1, 8, 3, 128, 100), nat.FTX_ERR_INVALID), ((1, 1, 8, 4, 96, 100), nat.FTX_ERR_UNSUPPORTED),
                        ((-1, 1, 8, 4, 128, 100), nat.FTX_ERR_INVALID), ((1, 1, 0, 1, 128, 100), nat.FTX_ERR_INVALID),
                        ((1, 1, 8, 4, 128, -1), nat.FTX_ERR_INVALID), ((1 << 25, 1, 1, 1, 64, 1), nat.FTX_ERR_INVALID),
                        ((1 << 24, 1 << 24, 65536, 1, 64, 1), nat.FTX_ERR_INVALID),
                        ((1 << 24, 1, 64, 64, 64, 1 << 20), nat.FTX_ERR_UNSUPPORTED)):
        assert work(*shape, ctypes.byref(b)) == code, shape
    assert work(0, 1, 8, 4, 128, 100, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert work(1, 1, 8, 4, 128, 0, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert work(1, 1, 8, 8, 128, 32000, ctypes.byref(b)) == nat.FTX_OK and b.value > 0
    assert work(1, 1, 8, 8, 128, 32000, None) == nat.FTX_ERR_INVALID

    def cache(**change):
        c = nat.Kv8Cache(0, 0, 4, 0, 2, 0, 0, 2, 2, 64, 128, nat.KV8_INT8)
        for k, v in change.items():
            setattr(c, k, v)
        return ctypes.byref(c)

    def attend(c, b=1, t=1, h=4, scale=1.0):
        return lib.ftx_kv8_attention(c, nul, nul, b, t, h, (ctypes.c_int64 * 6)(), scale, 100, nul, 0, nul)

    assert attend(None) == nat.FTX_ERR_INVALID
    for change in ({"d": 96}, {"page_tokens": 48}, {"page_tokens": 16}, {"page_tokens": 8192}, {"pages": 0},
                   {"kv_heads": 3}, {"kv_heads": 0}, {"format": 2}, {"width": -1}, {"table_stride": 1},
                   {"width": 1 << 30, "table_stride": 1 << 30}):
        assert attend(cache(**change)) in (nat.FTX_ERR_INVALID, nat.FTX_ERR_UNSUPPORTED), change
    assert attend(cache(), scale=0.0) == attend(cache(), scale=float("nan")) == nat.FTX_ERR_INVALID
    assert attend(cache(), b=0) == nat.FTX_OK and attend(cache(), t=0) == nat.FTX_OK
    assert attend(cache()) == nat.FTX_ERR_INVALID and b"null" in lib.ftx_last_error()
    assert lib.ftx_kv8_append(cache(), nul, nul, nul, nul, nul, -1, nul, 1, 1, 4, (ctypes.c_int64 * 9)(), nul) == \
        nat.FTX_ERR_INVALID
    assert lib.ftx_kv8_append(cache(), nul, nul, nul, nul, nul, 8, nul, 0, 1, 4, nul, nul) == nat.FTX_OK

    def copy(src, dst, pages=4, layers=1, d=64):
        n = len(src)
        return lib.ftx_kv8_copy_pages(nul, nul, layers, pages, 1, 32, d, (ctypes.c_int32 * n)(*src),
                                      (ctypes.c_int32 * n)(*dst), n, nul)

    assert copy([], []) == nat.FTX_OK and copy([0], [1], layers=0) == nat.FTX_OK
    for src, dst in (([0], [4]), ([-1], [0]), ([4], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0])):
        assert copy(src, dst) == nat.FTX_ERR_INVALID, (src, dst)
    assert copy([0], [1], d=80) == nat.FTX_ERR_UNSUPPORTED
    assert copy([0], [1]) == nat.FTX_ERR_INVALID and b"null" in lib.ftx_last_error()

    size = lib.ftx_int8_matmul_workspace
    for shape, code in (((1, 1, 24), nat.FTX_ERR_UNSUPPORTED), ((1, 1, 131088), nat.FTX_ERR_UNSUPPORTED),
                        ((-1, 1, 16), nat.FTX_ERR_INVALID), ((1 << 24, 1, 16), nat.FTX_ERR_INVALID),
                        ((1, (1 << 24) + 1, 16), nat.FTX_ERR_INVALID)):
        assert size(*shape, ctypes.byref(b)) == code, shape
    assert size(0, 64, 64, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert size(1, 64, 64, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert size(40, 4096, 4096, ctypes.byref(b)) == nat.FTX_OK and b.value > 0
    parts = b.value
    assert lib.ftx_int8_linear_workspace(40, 4096, 4096, ctypes.byref(b)) == nat.FTX_OK
    assert b.value == 40 * 4096 + 256 + parts
    assert lib.ftx_int8_quantize(nul, 24, nul, nul, 2, 32, nul) == nat.FTX_ERR_INVALID  # rows that overlap
    assert lib.ftx_int8_quantize(nul, 32, nul, nul, 0, 32, nul) == nat.FTX_OK
    assert lib.ftx_int8_matmul(nul, nul, nul, nul, nul, 0, 5, 32, nul, 0, nul) == nat.FTX_OK
    assert lib.ftx_int8_linear(nul, 32, nul, nul, nul, 1, 5, 32, nul, 0, nul) == nat.FTX_ERR_INVALID


def test_int8_linear_on_the_host_is_the_definition():
    torch.manual_seed(0)
    lin = W.init_normal_(W.Int8Linear(48, 10), seed=3)
    assert lin.weight.dtype == torch.int8 and int(lin.weight.abs().max()) == 127
    x = torch.randn(3, 5, 48).bfloat16()
    x[0, 0] = 0.0
    codes = (x.double() / (x.double().abs().amax(-1, keepdim=True) / 127)).round().nan_to_num(0.0)
    want = (codes @ lin.weight.double().t()) * (x.double().abs().amax(-1, keepdim=True) / 127) * lin.scale.double()
    assert ((lin(x).double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-12).all()
    shape = W.LlamaShape(n_layers=1, hidden=64, n_heads=2, n_kv_heads=1, head_dim=32, inter=96, int8=True)
    layer = W.DecoderLayer(shape, torch.bfloat16)
    assert sum(p.numel() * p.element_size() for p in layer.parameters()) == shape.layer_bytes()


def test_a_missing_torch_binding_fails_loudly(monkeypatch):
    import sys

    import flextensor_amd
    from flextensor_amd import _native as nat

    monkeypatch.setattr(nat, "_torch_calls", None)
    monkeypatch.delattr(flextensor_amd, "_ftx_torch", raising=False)
    monkeypatch.setitem(sys.modules, "flextensor_amd._ftx_torch", None)
    with pytest.raises(nat.FtxLibraryMissing, match="torch binding"):
        nat.torch_calls()


def test_the_torch_binding_leaves_what_it_does_not_know_alone():
    from flextensor_amd import _native as nat

    calls = nat.torch_calls()
    t = torch.zeros(2, 2, 2, 64, dtype=torch.bfloat16)
    for name, n in (("append", 12), ("attention", 10), ("copy_pages", 6), ("int8_linear", 5), ("int8_matmul", 6)):
        call = getattr(calls, name)
        for args in ((), (None,) * n, (t,) * (n - 2) + (0, 0), ([],) * (n - 2) + (0, 0)):  # too few, no tensors, the host's
            assert call(*args) is None
