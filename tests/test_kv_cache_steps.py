"""Steps of the paged cache that are not committed at once: what they reserve is theirs alone, and what a step may
count. The binding that its calls go through. Without a GPU."""

from __future__ import annotations

import random
import shutil
import subprocess
import sys

import pytest
import torch

from flextensor_amd import _native as nat
from flextensor_amd import kv_cache as kvc
from flextensor_amd import workloads as W

PAGE = 32


@pytest.fixture
def pool(monkeypatch):
    """A pool whose page copies are torch's."""

    def copy(codes, scales, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        codes.view(torch.uint8)[:, dst] = codes.view(torch.uint8)[:, src]
        scales[:, dst] = scales[:, src]

    monkeypatch.setattr(kvc, "copy_pages", copy)
    return kvc.PagedKVCache(1, 1, 64, 16, page_tokens=PAGE, dtype=torch.int8, device="cpu")


def _written(cache, step):
    """The pages that a step's appends write, by its own table."""
    pages = []
    for row, start, count in zip(step.table.tolist(), step.starts.tolist(), step.new.tolist()):
        if count:
            pages += row[start // PAGE: (start + count - 1) // PAGE + 1]
    return pages


def test_a_fork_between_begin_and_commit_holds_committed_tokens_alone(pool):
    a = pool.open()
    step = pool.begin([a], 40)
    b = pool.fork(a)
    assert pool.table(b) == [] and pool.length(b) == 0
    pool.commit(step)
    other = pool.begin([b], 40)
    assert not set(pool.table(a)) & set(_written(pool, other))


def test_a_fork_shares_the_page_in_use_and_none_that_is_reserved(pool):
    a = pool.open()
    pool.commit(pool.begin([a], 10))
    step = pool.begin([a], 100)
    b = pool.fork(a)
    assert pool.table(b) == pool.table(a)[:1]
    pool.commit(step)
    other = pool.begin([b], 100)
    assert not set(pool.table(a)) & set(_written(pool, other)) and pool.table(a) == step.table[0].tolist()


def test_forks_after_an_abandoned_step_write_pages_of_their_own(pool):
    a = pool.open()
    pool.begin([a], 100)  # a pass that failed
    pool.commit(pool.begin([a], 10))
    b = pool.fork(a)
    step = pool.begin([a, b], 40)
    pages = _written(pool, step)
    assert len(pages) == 4 and len(set(pages)) == 4


def test_every_shared_page_that_a_step_writes_is_copied(pool):
    """Held pages past the one in use, however they came to be shared."""
    a = pool.open()
    pool.begin([a], 100)
    b = pool.open()
    pool._pages[b] = list(pool._pages[a])
    for p in pool._pages[a]:
        pool._refs[p] += 1
    step = pool.begin([a, b], 70)
    pages = _written(pool, step)
    assert len(pages) == 6 and len(set(pages)) == 6
    assert all(pool._refs[p] == 1 for p in pages)


def test_a_long_run_with_steps_in_flight(pool):
    """Random forks, truncations and closings between begin and commit, and steps that are given up: no page that a
    step writes is held by another sequence when it begins, none that holds another's committed tokens is written."""
    rng = random.Random(11)
    held: list[int] = []
    flight = []
    for _ in range(1500):
        move = rng.choice(["open", "begin", "begin", "commit", "fork", "fork", "truncate", "close", "give up"])
        busy = {s for step in flight for s in step.sequences}
        idle = [s for s in held if s not in busy]
        try:
            if move == "open" and len(held) < 6:
                held.append(pool.open())
            elif move == "begin" and idle:
                some = rng.sample(idle, rng.randint(1, len(idle)))
                step = pool.begin(some, [rng.randint(0, 70) for _ in some])
                pages = _written(pool, step)
                assert len(set(pages)) == len(pages) and all(pool._refs[p] == 1 for p in pages)
                flight.append(step)
            elif move == "commit" and flight:
                pool.commit(flight.pop(rng.randrange(len(flight))))
            elif move == "give up" and flight:
                flight.pop(rng.randrange(len(flight)))
            elif move == "fork" and held and len(held) < 8:
                held.append(pool.fork(rng.choice(held)))
            elif move == "truncate" and idle:
                s = rng.choice(idle)
                pool.truncate(s, rng.randint(0, pool.length(s)))
            elif move == "close" and idle:
                s = rng.choice(idle)
                pool.close(s)
                held.remove(s)
        except kvc.KVCacheFull:
            pass
        for step in flight:  # committed tokens of a sequence stay out of the reach of the steps of others
            for s, row, start, count in zip(step.sequences, step.table.tolist(), step.starts.tolist(), step.new.tolist()):
                for at in range(start // PAGE, -(-(start + count) // PAGE)) if count else ():
                    for other in held:
                        if other != s and row[at] in pool.table(other):
                            assert pool.table(other).index(row[at]) == at and pool.length(other) <= start


def test_a_copy_that_fails_changes_nothing(pool, monkeypatch):
    a = pool.open()
    pool.commit(pool.begin([a], 10))
    b = pool.fork(a)
    before = pool.table(a), pool.table(b), list(pool._refs), list(pool._free)

    def fails(*args):
        raise RuntimeError("no copy")

    with monkeypatch.context() as m:
        m.setattr(kvc, "copy_pages", fails)
        with pytest.raises(RuntimeError, match="no copy"):
            pool.begin([a, b], 1)
    assert (pool.table(a), pool.table(b), pool._refs, pool._free) == before
    pages = _written(pool, pool.begin([a, b], 1))
    assert len(set(pages)) == 2


def test_a_step_is_counted_once(pool):
    a, b = pool.open(), pool.open()
    step = pool.begin([a, b], [10, 0])
    pool.commit(step)
    with pytest.raises(ValueError, match="committed before"):
        pool.commit(step)
    assert pool.length(a) == 10 and pool.length(b) == 0


def test_a_step_of_sequences_that_changed_is_not_counted(pool):
    a, b = pool.open(), pool.open()
    pool.commit(pool.begin([a, b], 40))

    def refused(step):
        lengths = dict(pool._lengths)
        with pytest.raises(ValueError, match="changed"):
            pool.commit(step)
        assert pool._lengths == lengths

    step = pool.begin([b, a], 3)
    pool.truncate(a, 20)
    refused(step)  # of neither of its sequences
    step = pool.begin([a], 3)
    c = pool.fork(a)
    pool.begin([a], 3)  # writes a copy of the page that the first step would write
    refused(step)
    step = pool.begin([c], 3)
    pool.close(c)
    refused(step)
    refused(kvc.PagedKVCache(1, 1, 64, 4, page_tokens=PAGE, dtype=torch.int8, device="cpu").begin([], []))
    first, second = pool.begin([b], 3), pool.begin([b], 3)  # the same tokens again, in the same pages
    pool.commit(second)
    refused(first)
    assert pool.length(b) == 43


def test_a_compaction_after_the_pass_keeps_its_step(pool):
    a, b = pool.open(), pool.open()
    pool.commit(pool.begin([a], 40))
    step = pool.begin([b], 40)
    pool.close(a)
    assert pool.compact() == 2
    pool.commit(step)
    assert pool.length(b) == 40 and pool.table(b) == [0, 1]
    with pytest.raises(ValueError, match="committed before"):
        pool.commit(step)


def test_a_pass_holds_the_tokens_of_its_step_within_the_models_positions():
    """Refused before anything is written, by the model and by a layer's append."""
    shape = W.LlamaShape(n_layers=1, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, inter=96, vocab=50, max_seq=48)
    model = W.build_llama(shape, seed=0)
    cache = model.init_paged_cache(8, 32, torch.int8, "cpu")
    a, b = cache.open(), cache.open()
    cache.commit(cache.begin([a, b], [40, 3]))

    def refused(step, b, t, match):
        x = torch.zeros(b, t, 1, 64, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match=match):
            model(torch.zeros(b, t, dtype=torch.long), step=step)
        with pytest.raises(ValueError, match=match):
            step.layer(0).append(x, x, x, model.rope_cos, model.rope_sin)

    refused(cache.begin([a], 9), 1, 9, "48 positions")
    refused(cache.begin([b, a], [1, 9]), 2, 9, "48 positions")
    refused(cache.begin([a], 8), 1, 7, "the pass has 7 of 1")  # a row narrower than the tokens that commit would count
    refused(cache.begin([a], 8), 2, 8, "the pass has 8 of 2")
    refused(cache.begin([a, b], 1), 1, 1, "the pass has 1 of 1")
    # up to the last position, in rows wider than the step's, beside a sequence that adds nothing: only the host's
    # tensors are wrong
    for step, shape in ((cache.begin([a], 8), (1, 12)), (cache.begin([a, b], [0, 45]), (2, 45))):
        refused(step, *shape, "current GPU")


def test_the_torch_binding_takes_the_library_that_is_loaded(tmp_path):
    """A library loaded from another place is the only one in the process, and the binding's calls end in it."""
    other = tmp_path / "libftx_elsewhere.so"
    shutil.copy(nat.LIB_PATH, other)
    code = f"""
from flextensor_amd import _native as nat
nat.load({str(other)!r})
calls = nat.torch_calls()
maps = open("/proc/self/maps").read()
assert {str(other)!r} in maps and {nat.LIB_PATH.name!r} not in maps
assert calls.append(*[None] * 12) is None
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=nat.LIB_PATH.parent.parent)


def test_the_torch_binding_refuses_calls_before_it_has_a_library():
    code = """
import torch
from flextensor_amd import _ftx_torch
for call in (lambda: _ftx_torch.append(), lambda: _ftx_torch.use(0), lambda: _ftx_torch.use(None)):
    try:
        call()
    except (RuntimeError, ValueError, TypeError):
        continue
    raise SystemExit("not refused")
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=nat.LIB_PATH.parent.parent)


def test_a_page_list_too_long_for_the_memory_left_is_an_error():
    """Of the C entry, which no exception may leave: a list that takes hundreds of MiB to check where 128 are left."""
    code = """
import ctypes, resource
from flextensor_amd import _native as nat
lib = nat.load()
n = 20_000_000
src, dst = ((ctypes.c_int32 * n)() for _ in range(2))
import numpy as np
np.frombuffer(dst, dtype=np.int32)[:] = np.arange(1, n + 1, dtype=np.int32)
size = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (size + (128 << 20),) * 2)
rc = lib.ftx_kv8_copy_pages(None, None, 1, n + 1, 1, 32, 64, src, dst, n, None)
assert rc == nat.FTX_ERR_OOM, rc
assert b"page copy" in lib.ftx_last_error()
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120, cwd=nat.LIB_PATH.parent.parent)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_read_gives_zeros_for_holes(dtype):
    """Numbers outside the pool on either side, as a ragged step's table holds them: not the last page's tokens."""
    codes = torch.full((3, 2, 2, 1, 32 * 64), 5.0).to(dtype)
    codes.view(torch.uint8)[2] = 0x7F  # a NaN in e4m3
    scales = torch.full((3, 2, 2, 1), 2.0)
    table = torch.tensor([[0, -1], [3, 1], [1 << 30, -7]], dtype=torch.int32)
    for got in kvc.read(codes, scales, table):
        assert got.shape == (3, 64, 2, 64)
        assert (got[0, :32] == 10.0).all() and (got[1, 32:] == 10.0).all()
        assert not got[0, 32:].any() and not got[1, :32].any() and not got[2].any()


def test_a_step_of_no_sequences_is_an_empty_pass():
    shape = W.LlamaShape(n_layers=0, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, inter=96, vocab=50, max_seq=48)
    model = W.build_llama(shape, seed=0)
    cache = kvc.PagedKVCache(1, 1, 64, 4, page_tokens=PAGE, dtype=torch.int8, device="cpu")
    step = cache.begin([], [], tokens=3)
    assert model(torch.zeros(0, 3, dtype=torch.long), step=step).shape == (0, 1, 50)
    cache.commit(step)


@pytest.mark.parametrize("fails_at", ["the pool", "the prompts", "a step"])
def test_a_run_that_ends_early_leaves_no_sequences_behind(pool, monkeypatch, fails_at):
    shape = W.LlamaShape(n_layers=0, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, inter=96, vocab=50, max_seq=4096)
    model = W.build_llama(shape, seed=0)
    kept = pool.open()
    pool.commit(pool.begin([kept], 40))
    before, passes = pool.free_pages, []
    if fails_at != "the pool":
        forward = model.forward

        def fails(tokens, step):
            passes.append(step)
            if len(passes) == (1 if fails_at == "the prompts" else 3):
                raise RuntimeError("lost")
            return forward(tokens, step=step)

        monkeypatch.setattr(model, "forward", fails)
    prompts = [[1] * (400 if fails_at == "the pool" else 40)] * 2
    with pytest.raises((RuntimeError, kvc.KVCacheFull)):
        W.generate_paged(model, pool, prompts, 5, samples=2)
    assert pool.free_pages == before and list(pool._lengths) == [kept]
    monkeypatch.undo()
