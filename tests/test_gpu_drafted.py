"""Drafted decoding as a whole: tree passes over the paged cache against passes token by token, with 4-bit projections and
head norms, in ragged batches, in graphs, on other streams and streamed from host memory.

Two runs cache the same values under block scales that may differ, and add up in other orders. A block of normal values
in int8 is off by 0.9% of sigma and in e4m3 by 2.4% (rms); keys and values of two layers in each of the two runs add up
in quadrature to 2.5% and 6.8% of the logits. The bounds are three times that.
"""

from __future__ import annotations

import copy

import pytest
import torch

from flextensor_amd import hip
from flextensor_amd import kv_cache as kvc
from flextensor_amd import workloads as W
from flextensor_amd.config import OffloadConfig
from flextensor_amd.manager import OffloadManager, OffloadPhase

pytestmark = pytest.mark.gpu

BOUND = {torch.int8: 0.076, torch.float8_e4m3fn: 0.204}
SHAPE = W.LlamaShape(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, head_dim=64, inter=768, vocab=1000, max_seq=512,
                     int4=True, qk_norm=True)
PARENTS = [-1, 0, 0, 1, 2, 2, 5]


def _model(gpu, seed=1, **change):
    model = W.build_llama(W.LlamaShape(**{**SHAPE.__dict__, **change}), seed=seed)
    for layer in model.layers:
        if layer.attn.q_norm is not None:  # weights that let attention choose
            layer.attn.q_norm.weight.data.fill_(1.5)
            layer.attn.k_norm.weight.data.fill_(1.5)
    return model.to(gpu)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _prompts(*lengths):
    return [W.prompt_tokens(1, n, SHAPE.vocab, n)[0].tolist() for n in lengths]


def _prefill(model, cache, prompts, gpu):
    sequences = [cache.open() for _ in prompts]
    longest = max(map(len, prompts))
    tokens = torch.tensor([p + [0] * (longest - len(p)) for p in prompts], device=gpu)
    step = cache.begin(sequences, [len(p) for p in prompts])
    model(tokens, step=step)
    cache.commit(step)
    return sequences


def _chain(model, prompt, tokens, dtype, gpu):
    """The logits behind each of ``tokens``, one pass a token."""
    cache = model.init_paged_cache(12, 32, dtype, gpu)
    s = _prefill(model, cache, [prompt], gpu)
    rows = []
    for t in tokens:
        step = cache.begin(s, 1)
        rows.append(model(torch.tensor([[t]], device=gpu), step=step)[0, 0])
        cache.commit(step)
    return rows


@pytest.mark.parametrize("dtype", list(BOUND))
@pytest.mark.parametrize("change", [{}, {"head_dim": 128, "int4": False}, {"qk_norm": False}])
@pytest.mark.parametrize("levels", [False, True])
def test_each_path_of_a_tree_is_the_sequence_that_it_stands_for(gpu, dtype, change, levels):
    """All nodes at once or level by level; then the accepted path, and what follows it."""
    model = _model(gpu, **change)
    prompts = _prompts(61, 5, 130)
    nodes = W.prompt_tokens(3, len(PARENTS), SHAPE.vocab, 9).to(gpu)
    leaves = {3: [0, 1, 3], 4: [0, 2, 4], 6: [0, 2, 5, 6]}
    paths = [leaves[6], [0], leaves[4]]
    with torch.no_grad():
        cache = model.init_paged_cache(24, 32, dtype, gpu)
        sequences = _prefill(model, cache, prompts, gpu)
        tree = cache.draft(sequences, PARENTS)
        steps = tree.levels() if levels else [(0, len(PARENTS))]
        got = torch.cat([model(nodes[:, lo:hi], step=tree.nodes(lo, hi), every=True) for lo, hi in steps], 1)
        cache.accept(tree, paths)
        assert [cache.length(s) for s in sequences] == [len(p) + len(k) for p, k in zip(prompts, paths)]
        after = torch.tensor([[7], [8], [9]], device=gpu)
        step = cache.begin(sequences, 1)
        next_logits = model(after, step=step)
        for row, p in enumerate(prompts):
            for path in leaves.values():
                want = _chain(model, p, nodes[row, path].tolist(), dtype, gpu)
                for node, w in zip(path, want):
                    assert _rel(got[row, node], w) <= BOUND[dtype], (row, node)
            tokens = [*nodes[row, paths[row]].tolist(), int(after[row])]
            assert _rel(next_logits[row, 0], _chain(model, p, tokens, dtype, gpu)[-1]) <= BOUND[dtype]


@pytest.mark.parametrize("dtype", list(BOUND))
def test_drafted_decoding_is_greedy_decoding(gpu, dtype):
    """The tokens of a run token by token, up to one whose logit is as near the largest as the bound lets it be. A draft
    with the model's own weights is right almost always, another one seldom."""
    model = _model(gpu)
    prompts, steps = _prompts(45, 1, 100), 20
    cache = model.init_paged_cache(32, 32, dtype, gpu)
    _, want, logits = W.generate_paged(model, cache, prompts, steps)
    passes = {}
    for name, draft in (("itself", model), ("another", _model(gpu, seed=5, n_layers=1))):
        cache, draft_cache = (m.init_paged_cache(32, 32, dtype, gpu) for m in (model, draft))
        got, logps, passes[name] = W.generate_drafted(model, draft, cache, draft_cache, prompts, steps)
        assert cache.free_pages == draft_cache.free_pages == 32
        for row in range(len(prompts)):
            for i in range(steps):
                exact = logits[i][row, 0].double()
                off = BOUND[dtype] * float(exact.norm())
                a, b = int(want[row, i]), int(got[row, i])
                assert exact[a] - exact[b] <= 2 * off
                if a != b:
                    break
                assert abs(float(logps[row, i]) - float(exact.log_softmax(-1)[a])) <= 2 * off
    assert passes["itself"] < passes["another"] <= steps


def _operators(gpu, seed=0):
    """What one pass over drafted nodes calls, on its own tensors: inputs, and the calls as a function."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    b, n, h, kv, d, vocab = 3, 7, 8, 2, 128, 1000
    ang = torch.outer(torch.arange(400.0), 1.0 / 10000.0 ** (torch.arange(0, d, 2) / d))
    cos, sin = torch.cat([ang, ang], -1).cos().to(gpu), torch.cat([ang, ang], -1).sin().to(gpu)
    weight = torch.ones(d, device=gpu).bfloat16()
    sets = [1, 3, 5, 11, 21, 37, 101]
    depth = torch.tensor([0, 1, 1, 2, 2, 2, 3], dtype=torch.int32, device=gpu)
    tree = torch.tensor([sets], dtype=torch.int64, device=gpu).expand(b, n)
    table = torch.arange(30, dtype=torch.int32, device=gpu).view(b, 10)
    path = torch.tensor([[0, 2, 5, 6], [0, 1, 3, 0], [0, 0, 0, 0]], dtype=torch.int32, device=gpu)
    counts = torch.tensor([4, 3, 1], dtype=torch.int32, device=gpu)
    lin = W.init_normal_(W.Int4Linear(h * d, vocab), 4).to(gpu)
    tokens = torch.randint(0, vocab, (b, n), device=gpu, generator=g)

    def step(x, codes, scales, starts):
        q = kvc.append(x[:, :, :h], x[:, :, h: h + kv], x[:, :, h + kv:], cos, sin, codes[0], scales[0], table, starts,
                       positions=starts[:, None] + depth, q_norm=weight, k_norm=weight)
        o = kvc.tree_attention(q, codes[0], scales[0], table, starts, tree)
        logits = lin(o.view(b, n, h * d))
        scored = W.token_logprobs(logits, tokens, 4)
        kvc.keep(codes, scales, table, starts, path, counts)
        starts += counts
        return (o, logits, *scored)

    def state():
        codes = torch.zeros(1, 30, 2, kv, 1, 32 * d, dtype=torch.int8, device=gpu)
        starts = torch.tensor([0, 29, 290], dtype=torch.int32, device=gpu)
        return codes, torch.zeros(1, 30, 2, kv, 1, device=gpu), starts

    draws = [torch.randn(b, n, h + 2 * kv, d, device=gpu, generator=g).bfloat16() for _ in range(6)]
    return step, state, draws


def test_graph_replays_of_all_operators_are_the_eager_runs(gpu):
    """Positions that the graph itself advances; eager work and waits between the replays."""
    step, state, draws = _operators(gpu)
    want_state = state()
    want = [[t.clone() for t in step(x, *want_state)] for x in draws]
    held = state()
    x = draws[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, *held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, *held)
    for _ in range(2):
        for t, fresh in zip(held, state()):
            t.copy_(fresh)
        for draw, expected in zip(draws, want):
            x.copy_(draw)
            graph.replay()
            for a, e in zip(out, expected):
                assert torch.equal(a, e)
            torch.cuda.synchronize()
            step(draw, *state())
        for t, e in zip(held, want_state):
            assert torch.equal(t, e)


def test_two_captured_graphs_and_an_eager_run_do_not_share_workspaces(gpu):
    runs = [_operators(gpu, seed) for seed in (1, 2)]
    want, graphs = [], []
    for step, state, draws in runs:
        want.append([t.clone() for t in step(draws[0], *state())])
    torch.cuda.synchronize()
    for step, state, draws in runs:
        held = state()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(draws[0], *held)
        graphs.append((graph, held, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (_, state, _), (_, held, _) in zip(runs, graphs):
            for t, fresh in zip(held, state()):
                t.copy_(fresh)
        torch.cuda.synchronize()
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [step(draws[0], *state()) for step, state, draws in runs]
        torch.cuda.synchronize()
        for (_, _, out), again, expected in zip(graphs, eager, want):
            for a, b, e in zip(out, again, expected):
                assert torch.equal(a, e) and torch.equal(b, e)


def test_another_stream_gives_the_same_tokens(gpu):
    model, prompts = _model(gpu), _prompts(33, 64)
    caches = [model.init_paged_cache(12, 32, torch.int8, gpu) for _ in range(4)]
    want = W.generate_drafted(model, model, *caches[:2], prompts, 12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = W.generate_drafted(model, model, *caches[2:], prompts, 12)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[2] == want[2]


def test_a_streamed_4_bit_decoder_checks_drafts_as_the_resident_one(gpu):
    """Layers that stream from host memory, their 4-bit weights and head norms among them: the same tokens."""
    shape = W.LlamaShape(**{**SHAPE.__dict__, "n_layers": 4})
    model = W.build_llama(shape, seed=2)
    resident, draft = copy.deepcopy(model).to(gpu), _model(gpu, seed=3, n_layers=1)
    prompts = _prompts(50, 7)

    def run(m):
        cache, draft_cache = (r.init_paged_cache(12, 32, torch.int8, gpu) for r in (resident, draft))
        return W.generate_drafted(m, draft, cache, draft_cache, prompts, 6)

    want = run(resident)
    mgr = OffloadManager("drafted")
    try:
        mgr.offload(model, OffloadConfig(include_patterns=["layers.*"], num_blocks=2, min_blocks=2, discovery_iters=1,
                                         profiling_iters=1))
        for _ in range(3):  # discovery and profiling passes, then streamed ones
            got = run(model)
        assert mgr.phase == OffloadPhase.INFERENCE
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[2] == want[2]
    finally:
        mgr.release()


def test_scores_of_a_pass_are_those_of_the_logits(gpu):
    model = _model(gpu, qk_norm=False)
    model.init_cache(2, 128, gpu)
    tokens = W.prompt_tokens(2, 77, SHAPE.vocab).to(gpu)
    given, entropy, best, index = W.score(model, tokens, 5)
    with torch.no_grad():
        logits = model(tokens, every=True)[:, :-1].cpu()
    want = W.token_logprobs(logits.double(), tokens[:, 1:].cpu(), 5)
    assert torch.equal(index.cpu(), want[3])
    for a, b in ((given, want[0]), (entropy, want[1]), (best, want[2])):
        # sums of 1000 terms and logarithms of up to 7, each within a few 2^-23 of itself; the host's are fp32 too
        assert float((a.cpu().double() - b.double()).abs().max()) <= 2e-5


def test_4_bit_projections_follow_the_weights_they_stand_for(gpu):
    """Decode and prompt rows against the host form of the same codes: one rounding of the result and, from 17 rows on,
    one of each weight, both bf16."""
    for zeros in (False, True):
        lin = W.Int4Linear(512, 300, zeros)
        lin.quantize_(torch.randn(300, 512, generator=torch.Generator().manual_seed(0)) + 0.25)
        on_gpu = copy.deepcopy(lin).to(gpu)
        for shape in ((512,), (1, 1, 512), (5, 3, 512), (2, 40, 512), (0, 512)):
            x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).bfloat16()
            assert on_gpu.kernel_eligible(x.to(gpu)) == (x.numel() > 0)
            got, want = on_gpu(x.to(gpu)), lin(x)
            assert got.shape == want.shape and (not x.numel() or _rel(got.cpu(), want) <= 2.0 ** -7)
        x = torch.randn(4, 512, device=gpu).bfloat16().requires_grad_()
        y = on_gpu(x)  # a gradient goes through the weights
        y.backward(torch.ones_like(y))
        w = hip.int4_dequantize(lin.weight, lin.scale, lin.zero, 300, 512)
        # a sum of 300 fp32 products, rounded to bf16 once
        bound = 2.0 ** -8 * w.sum(0).abs() + 300 * 2.0 ** -24 * w.abs().sum(0)
        assert ((x.grad.cpu().double() - w.double().sum(0)).abs() <= bound.double()).all()


def test_head_norms_give_the_same_logits_with_both_caches(gpu):
    model = _model(gpu, int4=False)
    model.init_cache(1, 128, gpu)
    prompt = _prompts(70)
    with torch.no_grad():
        want = model(torch.tensor(prompt, device=gpu))
        cache = model.init_paged_cache(8, 32, torch.int8, gpu)
        s = [cache.open()]
        step = cache.begin(s, 70)
        got = model(torch.tensor(prompt, device=gpu), step=step)
        assert _rel(got, want) <= BOUND[torch.int8]
        # hooks on a norm are seen: it then runs by itself before the cache's launch
        seen = []
        hook = model.layers[1].attn.k_norm.register_forward_hook(lambda *a: seen.append(1))
        cache.commit(step)
        s2 = [cache.open()]
        step = cache.begin(s2, 70)
        again = model(torch.tensor(prompt, device=gpu), step=step)
        hook.remove()
        assert seen and _rel(again, got) <= BOUND[torch.int8]
