"""The decoder over a paged 8-bit cache and with int8 projections: against its dense bf16 form, in ragged batches,
forked, in graphs, on other streams and streamed from host memory.

A block of normal values quantised to int8 has its largest about four sigma out, so a step of 4 / 127 sigma and an
error of 0.9% of sigma; an e4m3 code is off by 2.4% of its value (rms of a relative error within 2^-4). Keys and
values of two layers add up in quadrature to 1.8% and 4.8% of the logits; the bounds are three times that.
"""

from __future__ import annotations

import copy

import pytest
import torch

from flextensor_amd import kv_cache as kvc
from flextensor_amd import workloads as W
from flextensor_amd.config import OffloadConfig
from flextensor_amd.manager import OffloadManager, OffloadPhase

pytestmark = pytest.mark.gpu

BOUND = {torch.int8: 0.054, torch.float8_e4m3fn: 0.144}
SAME_SUMS = 2.0 ** -5  # the same codes, sums in another order: bf16 roundings of two layers
SHAPE = W.LlamaShape(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, head_dim=64, inter=768, vocab=1000, max_seq=512)


def _model(gpu, **change):
    shape = W.LlamaShape(**{**SHAPE.__dict__, **change})
    return W.build_llama(shape, seed=1).to(gpu)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _prompt(n, seed=0):
    return W.prompt_tokens(1, n, SHAPE.vocab, seed)[0].tolist()


@pytest.mark.parametrize("dtype", list(BOUND))
@pytest.mark.parametrize("head_dim", [64, 128])
def test_paged_decoding_follows_the_dense_cache(gpu, dtype, head_dim):
    model = _model(gpu, head_dim=head_dim)
    prompt = _prompt(70)
    model.init_cache(1, 128, gpu)
    with torch.no_grad():
        tokens = torch.tensor([prompt], device=gpu)
        want = [model(tokens)]
        cache = model.init_paged_cache(8, 32, dtype, gpu)
        seq = cache.open()
        step = cache.begin([seq], len(prompt))
        got = [model(tokens, step=step)]
        cache.commit(step)
        for i in range(6):  # the dense run's tokens into both
            tok = want[-1].argmax(-1)
            want.append(model(tok, len(prompt) + i))
            step = cache.begin([seq], 1)
            got.append(model(tok, step=step))
            cache.commit(step)
    for a, b in zip(got, want):
        assert _rel(a, b) <= BOUND[dtype]
    keys, vals = kvc.read(cache.codes[1], cache.scales[1], torch.tensor(cache.table(seq), device=gpu))
    n = cache.length(seq)
    assert _rel(keys[:n], model.cache_k[1][0, :n]) <= BOUND[dtype]
    assert _rel(vals[:n], model.cache_v[1][0, :n]) <= BOUND[dtype]
    assert not keys[n:n + 32 - n % 32].any()  # the rest of the last block


def test_ragged_batches_give_each_sequence_its_own_answer(gpu):
    model = _model(gpu)
    prompts = [_prompt(n, n) for n in (45, 1, 100, 32)]
    cache = model.init_paged_cache(24, 32, torch.int8, gpu)
    _, tokens, logits = W.generate_paged(model, cache, prompts, 5)
    for i, p in enumerate(prompts):
        alone = model.init_paged_cache(8, 32, torch.int8, gpu)
        _, want_tokens, want = W.generate_paged(model, alone, [p], 5)
        assert _rel(logits[0][i], want[0][0]) <= SAME_SUMS
        if torch.equal(tokens[i], want_tokens[0]):  # greedy choices may part where two logits are near
            assert all(_rel(a[i], b[0]) <= SAME_SUMS for a, b in zip(logits, want))


def test_forked_samples_share_their_prompt(gpu):
    model = _model(gpu)
    prompts = [_prompt(40, 1), _prompt(64, 2)]
    cache = model.init_paged_cache(16, 32, torch.float8_e4m3fn, gpu)
    seqs, tokens, _ = W.generate_paged(model, cache, prompts, 4, samples=3)
    assert len(seqs) == 6 and len(set(tokens[:3, 0].tolist())) == 3
    assert len({cache.table(s)[0] for s in seqs[:3]}) == 1      # the full page is shared
    assert len({cache.table(s)[1] for s in seqs[:3]}) == 3      # the one in use is not
    assert len({tuple(cache.table(s)[:2]) for s in seqs[3:]}) == 1
    # what a fork has read and written is what the sequence alone would have
    alone = model.init_paged_cache(8, 32, torch.float8_e4m3fn, gpu)
    s = alone.open()
    with torch.no_grad():
        for chunk in ([prompts[0]], *[[[int(t)]] for t in tokens[1, :3]]):
            step = alone.begin([s], len(chunk[0]))
            model(torch.tensor(chunk, device=gpu), step=step)
            alone.commit(step)
    n = alone.length(s)
    assert n == cache.length(seqs[1])
    for layer in range(SHAPE.n_layers):
        for a, b in zip(*(kvc.read(c.codes[layer], c.scales[layer], torch.tensor(c.table(q), device=gpu))
                          for c, q in ((cache, seqs[1]), (alone, s)))):
            assert _rel(a[:n], b[:n]) <= BOUND[torch.float8_e4m3fn]
    for q in seqs:
        cache.close(q)
    assert cache.free_pages == cache.pages


def test_compaction_between_steps_changes_no_answer(gpu):
    model = _model(gpu)
    cache = model.init_paged_cache(20, 32, torch.int8, gpu)
    first = cache.open()
    step = cache.begin([first], 200)  # pages 0 .. 6, given back below
    cache.commit(step)
    prompt = _prompt(90)
    seq = cache.open()
    with torch.no_grad():
        step = cache.begin([seq], 90)
        logits = model(torch.tensor([prompt], device=gpu), step=step)
        cache.commit(step)
        tok = logits.argmax(-1)
        step = cache.begin([seq], 1)
        want = model(tok, step=step)  # not committed: the next step writes the same token again
        cache.close(first)
        assert cache.compact() == 3 and cache.table(seq) == [0, 1, 2]
        cache.resize(4)
        step = cache.begin([seq], 1)
        got = model(tok, step=step)
    assert torch.equal(got, want)


def test_graph_replays_follow_the_device_positions(gpu):
    """A captured append and attention advance with the starts that the graph itself counts; eager work between the
    replays; each replay's bits are the eager run's."""
    g = torch.Generator(device=gpu).manual_seed(0)
    b, h, kv, d, page = 3, 8, 2, 128, 32
    ang = torch.outer(torch.arange(400.0), 1.0 / 10000.0 ** (torch.arange(0, d, 2) / d))
    cos, sin = torch.cat([ang, ang], -1).cos().to(gpu), torch.cat([ang, ang], -1).sin().to(gpu)
    table = torch.arange(30, dtype=torch.int32, device=gpu).view(b, 10)

    def pool():
        codes = torch.zeros(30, 2, kv, 1, 32 * d, dtype=torch.int8, device=gpu)
        return codes, torch.zeros(30, 2, kv, 1, device=gpu)

    starts0 = torch.tensor([0, 29, 290], dtype=torch.int32, device=gpu)
    draws = [torch.randn(b, 1, h + 2 * kv, d, device=gpu, generator=g).bfloat16() for _ in range(6)]

    def step(x, codes, scales, starts):
        q = kvc.append(x[:, :, :h], x[:, :, h: h + kv], x[:, :, h + kv:], cos, sin, codes, scales, table, starts)
        return kvc.attention(q, codes, scales, table, starts)

    codes, scales = pool()
    starts = starts0.clone()
    want = []
    for x in draws:
        want.append(step(x, codes, scales, starts))
        starts += 1
    want_codes, want_scales = codes.clone(), scales.clone()

    codes, scales = pool()
    starts = starts0.clone()
    x = draws[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, codes, scales, starts)
    torch.cuda.current_stream().wait_stream(side)
    codes.zero_()
    scales.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, codes, scales, starts)
        starts += 1
    codes.zero_()
    scales.zero_()
    starts.copy_(starts0)
    for draw, expected in zip(draws, want):
        x.copy_(draw)
        graph.replay()
        assert torch.equal(out, expected)
        torch.cuda.synchronize()
        torch.ones(1000, device=gpu).sum()
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)


def test_another_stream_gives_the_same_bits(gpu):
    model = _model(gpu, int8=True)
    prompts = [_prompt(33), _prompt(64, 3)]
    want_cache = model.init_paged_cache(8, 32, torch.int8, gpu)
    _, want, want_logits = W.generate_paged(model, want_cache, prompts, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache = model.init_paged_cache(8, 32, torch.int8, gpu)
        _, got, logits = W.generate_paged(model, cache, prompts, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(logits, want_logits))


def test_int8_projections_follow_the_weights_they_stand_for(gpu):
    """Decode and prompt rows of a decoder layer against the torch form of the same codes: bf16 roundings apart."""
    model = _model(gpu, int8=True)
    layer = model.layers[0]
    for rows in (1, 40):
        x = torch.randn(1, rows, SHAPE.hidden, device=gpu, generator=torch.Generator(device=gpu).manual_seed(rows))
        x = x.bfloat16()
        for lin in (layer.attn.wq, layer.gate):
            want = copy.deepcopy(lin).cpu()(x.cpu())
            assert _rel(lin(x).cpu(), want) <= 2.0 ** -8
        grouped = W.int8_group(x, [layer.attn.wq, layer.attn.wk])
        assert torch.equal(grouped[0], layer.attn.wq(x)) and torch.equal(grouped[1], layer.attn.wk(x))


@pytest.mark.parametrize("int8", [True, False])
def test_streamed_decoder_over_a_paged_cache_is_the_resident_one(gpu, int8):
    """Layers that stream from host memory, int8 weights among them, with the cache on the GPU: the same bits."""
    shape = W.LlamaShape(**{**SHAPE.__dict__, "n_layers": 4, "int8": int8})
    model = W.build_llama(shape, seed=2)
    resident = copy.deepcopy(model).to(gpu)
    prompts = [_prompt(50), _prompt(7, 9)]
    want_cache = resident.init_paged_cache(12, 32, torch.int8, gpu)
    _, want, want_logits = W.generate_paged(resident, want_cache, prompts, 4)
    mgr = OffloadManager("paged")
    try:
        mgr.offload(model, OffloadConfig(include_patterns=["layers.*"], num_blocks=2, min_blocks=2, discovery_iters=1,
                                         profiling_iters=1))
        for _ in range(3):  # discovery and profiling passes, then streamed ones
            cache = resident.init_paged_cache(12, 32, torch.int8, gpu)
            _, got, logits = W.generate_paged(model, cache, prompts, 4)
        assert mgr.phase == OffloadPhase.INFERENCE
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(logits, want_logits))
    finally:
        mgr.release()
