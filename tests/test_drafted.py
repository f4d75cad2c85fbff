"""Drafted trees of the paged cache, decoding with them, log probabilities and the 4-bit projection as a module. Without
a GPU: page moves are torch's."""

from __future__ import annotations

import ctypes

import pytest
import torch

from flextensor_amd import _native as nat
from flextensor_amd import hip
from flextensor_amd import kv_cache as kvc
from flextensor_amd import workloads as W

PAGE = 32


@pytest.fixture
def kept(monkeypatch):
    """The calls of the operator that moves the accepted nodes."""
    calls = []

    def copy(codes, scales, src, dst):
        codes.view(torch.uint8)[:, dst] = codes.view(torch.uint8)[:, src]
        scales[:, dst] = scales[:, src]

    monkeypatch.setattr(kvc, "copy_pages", copy)
    monkeypatch.setattr(kvc, "keep", lambda codes, scales, *ints: calls.append([x.tolist() for x in ints]))
    return calls


def _pool(pages=16):
    return kvc.PagedKVCache(1, 1, 64, pages, page_tokens=PAGE, dtype=torch.int8, device="cpu")


def _grown(cache, *lengths):
    sequences = [cache.open() for _ in lengths]
    cache.commit(cache.begin(sequences, list(lengths)))
    return sequences


def test_a_tree_knows_its_nodes_ancestors_and_positions():
    cache = _pool()
    a, b = _grown(cache, 30, 5)
    tree = cache.draft([a, b], [-1, 0, 0, 1, 2, -1])
    assert tree.depths == (0, 1, 1, 2, 2, 0)
    assert tree.sets.tolist() == [[0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100000]]
    assert tree.positions.tolist() == [[30, 31, 31, 32, 32, 30], [5, 6, 6, 7, 7, 5]]
    assert tree.starts.tolist() == [[30 + i, 5 + i] for i in range(6)]
    assert len(cache.table(a)) == 2 and len(cache.table(b)) == 1 and cache.length(a) == 30
    with pytest.raises(ValueError, match="level by level"):
        tree.levels()
    assert cache.draft([a], [-1, 0, 0, 1, 1, 3]).levels() == [(0, 1), (1, 3), (3, 5), (5, 6)]


def test_a_tree_of_64_nodes_uses_every_bit():
    cache = _pool()
    tree = cache.draft(_grown(cache, 3), list(range(-1, 63)))
    assert tree.sets[0, 63] == -1 and tree.sets[0, 62] == 2 ** 63 - 1 and tree.depths[63] == 63


@pytest.mark.parametrize("parents", [[], [0], [-1, 1], [-1, -2], [-1] * 65])
def test_what_is_no_tree_is_refused(parents):
    cache = _pool()
    s, = _grown(cache, 3)
    with pytest.raises(ValueError, match="nodes, each behind its parent"):
        cache.draft([s], parents)
    assert len(cache.table(s)) == 1


def test_accepted_paths_are_moved_and_counted(kept):
    cache = _pool()
    a, b, c = _grown(cache, 30, 64, 7)
    tree = cache.draft([a, b, c], [-1, 0, 0, 1, 2, 4])
    cache.accept(tree, [[0, 2, 4, 5], [], [0, 1]])
    assert [cache.length(s) for s in (a, b, c)] == [34, 64, 9]
    table, starts, path, counts = kept[0]
    assert starts == [30, 64, 7] and counts == [4, 0, 2] and path == [[0, 2, 4, 5], [0] * 4, [0, 1, 0, 0]]
    assert [[p for p in row if p >= 0] for row in table] == [cache.table(s) for s in (a, b, c)]
    with pytest.raises(ValueError, match="committed before"):
        cache.accept(tree, [[0], [0], [0]])


def test_paths_that_are_where_they_belong_move_nothing(kept):
    cache = _pool()
    a, b = _grown(cache, 30, 64)
    cache.accept(cache.draft([a, b], [-1, 0, 0]), [[0, 1], []])
    assert not kept and cache.length(a) == 32 and cache.length(b) == 64
    cache.accept(cache.draft([], [-1]), [])


@pytest.mark.parametrize("path", [[1], [0, 3], [0, 1, 2], [2, 0], [0, 6], [-1], [0, 0]])
def test_what_is_no_path_is_refused(kept, path):
    cache = _pool()
    a, b = _grown(cache, 30, 4)
    tree = cache.draft([a, b], [-1, 0, 0, 1, 2, 4])
    with pytest.raises(ValueError, match="no path"):
        cache.accept(tree, [[0], path])
    with pytest.raises(ValueError, match="1 paths for 2"):
        cache.accept(tree, [[0]])
    assert not kept and cache.length(a) == 30


def test_a_tree_of_sequences_that_changed_is_not_accepted(kept):
    cache = _pool()
    a, b = _grown(cache, 30, 4)
    tree = cache.draft([a, b], [-1, 0, 0])
    cache.truncate(a, 20)
    with pytest.raises(ValueError, match="changed"):
        cache.accept(tree, [[0, 2], [0]])
    tree = cache.draft([a, b], [-1, 0, 0])
    cache.close(b)
    with pytest.raises(ValueError, match="changed"):
        cache.accept(tree, [[0, 2], [0]])
    assert not kept


def test_a_compaction_between_draft_and_accept_moves_the_new_pages(kept):
    cache = _pool()
    first, a = _grown(cache, 100, 30)
    tree = cache.draft([a], [-1, 0, 0, 2])
    old = cache.table(a)
    cache.close(first)
    assert cache.compact() and cache.table(a) != old
    cache.accept(tree, [[0, 2, 3]])
    assert kept[0][0] == [cache.table(a)] and cache.length(a) == 33


def test_a_pool_too_small_for_a_tree_changes_nothing():
    cache = _pool(2)
    a, b = _grown(cache, 30, 30)
    with pytest.raises(kvc.KVCacheFull):
        cache.draft([a, b], [-1, 0, 0])
    assert cache.length(a) == 30 and len(cache.table(a)) == 1


def test_a_pass_holds_the_nodes_of_its_tree_within_the_models_positions():
    cache = _pool()
    s = _grown(cache, 30, 4)
    tree = cache.draft(s, [-1, 0, 0, 1])
    tree.nodes().check(2, 4, 33)
    tree.nodes(1, 3).check(2, 2, 32)
    for bad in ((1, 4, 33), (2, 3, 33), (2, 5, 33), (2, 4, 32)):
        with pytest.raises(ValueError):
            tree.nodes().check(*bad)
    for first, last in ((0, 0), (2, 1), (0, 5), (-1, 2)):
        with pytest.raises(ValueError, match="of a tree of 4"):
            tree.nodes(first, last)


def _bigram(seed):
    """A model whose next token depends on the last one alone."""
    shape = W.LlamaShape(n_layers=0, hidden=64, n_heads=1, n_kv_heads=1, head_dim=64, inter=96, vocab=50, max_seq=4096)
    return W.build_llama(shape, seed=seed)


@pytest.mark.parametrize("parents", [(-1,), (-1, 0), (-1, 0, 0, 0), W.DRAFT_TREE])
@pytest.mark.parametrize("same", [True, False])
def test_drafted_tokens_are_the_greedy_ones(kept, parents, same):
    model, steps = _bigram(0), 17
    draft = model if same else _bigram(1)
    prompts = [[3], [4, 5, 6], [7] * 40]
    cache, draft_cache = _pool(), _pool()
    with torch.no_grad():
        logits = model(torch.arange(50)[:, None]).squeeze(1)
    want, logps = [], []
    for p in prompts:
        token, row = p[-1], []
        for _ in range(steps):
            logps.append(float(logits[token].log_softmax(-1).max()))
            token = int(logits[token].argmax())
            row.append(token)
        want.append(row)
    got, logp, passes = W.generate_drafted(model, draft, cache, draft_cache, prompts, steps, parents)
    assert got.tolist() == want
    # one bf16 product either way; the sums of 50 exponentials in fp32 in another order
    assert torch.allclose(logp.flatten().double(), torch.tensor(logps).double(), atol=1e-5)
    deepest = 1 + max(sum(1 for _ in _ancestors(parents, i)) for i in range(len(parents)))
    if same:  # every pass keeps the longest chain
        assert passes == 1 + -(-(steps - 1) // deepest)
    assert passes <= steps and cache.free_pages == cache.pages == draft_cache.free_pages


def _ancestors(parents, node):
    while parents[node] >= 0:
        node = parents[node]
        yield node


@pytest.mark.parametrize("parents", [(), (0,), (-1, -1), (-1, 0, 1, 0)])
def test_trees_that_decoding_cannot_use_are_refused(kept, parents):
    model, cache = _bigram(0), _pool()
    with pytest.raises(ValueError, match="one root|level by level"):
        W.generate_drafted(model, model, cache, _pool(), [[3]], 5, parents)
    assert cache.free_pages == cache.pages and not cache._lengths


def test_log_probabilities_of_the_host():
    torch.manual_seed(0)
    logits = torch.randn(2, 3, 20)
    logits[0, 0, 3:] = float("-inf")
    logits[1, 2, 7] = logits[1, 2, 4] = 9.0
    tokens = torch.tensor([[1, 19, -1], [5, 20, 4]])
    given, entropy, best, index = W.token_logprobs(logits, tokens, 3)
    want = logits.double().log_softmax(-1)
    assert given.shape == entropy.shape == (2, 3) and best.shape == index.shape == (2, 3, 3)
    # a term of the sum is off by 2^-24 of itself, a logarithm by 2^-23 of up to 5
    assert abs(given[0, 0] - want[0, 0, 1]) <= 1e-6 and abs(given[0, 1] - want[0, 1, 19]) <= 1e-6
    assert given[0, 2] == 0 and given[1, 1].isnan() and index[1, 2, :2].tolist() == [4, 7]
    assert torch.allclose(best.double(), want.topk(3).values, atol=1e-6)
    ent = -(want.exp() * want.nan_to_num(neginf=0.0)).sum(-1)
    assert torch.allclose(entropy.double(), ent, atol=1e-5)
    assert [x.shape for x in W.token_logprobs(logits[:0], tokens[:0])] == [(0, 3), (0, 3), (0, 3, 0), (0, 3, 0)]


def test_a_score_is_what_each_token_is_given_by_the_ones_before():
    shape = W.LlamaShape(n_layers=2, hidden=64, n_heads=2, n_kv_heads=1, head_dim=32, inter=96, vocab=50, max_seq=64,
                         qk_norm=True)
    model = W.build_llama(shape, seed=0)
    model.init_cache(2, 16, torch.device("cpu"))
    tokens = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(0))
    given, entropy, best, index = W.score(model, tokens, 2)
    assert given.shape == (2, 8) and index.shape == (2, 8, 2)
    with torch.no_grad():
        for i in range(1, 9):
            logp = model(tokens[:, :i]).squeeze(1).double().log_softmax(-1)
            # the same bf16 operations on other shapes; logits of about 0.2 are off by bf16 steps of 2^-11
            assert torch.allclose(given[:, i - 1].double(), logp.gather(1, tokens[:, i: i + 1])[:, 0], atol=0.01)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("k, group", [(256, 128), (192, 64), (96, 32)])
def test_a_4_bit_projection_takes_the_nearest_weights(k, group, zeros):
    torch.manual_seed(1)
    lin = W.Int4Linear(k, 21, zeros)
    assert lin.scale.shape[3] == 128 // group
    w = torch.randn(21, k) + 0.5
    lin.quantize_(w)
    got = hip.int4_dequantize(lin.weight, lin.scale, lin.zero, 21, k)
    grouped = w.unflatten(1, (-1, group))
    # half a step of the scale, which bf16 rounds by 2^-8 (times 7 or 15 steps), and a zero that it rounds by as much
    if zeros:
        step = (grouped.amax(-1) - grouped.amin(-1)) / 15
        bound = step * (0.5 + 15 * 2.0 ** -8 + 15 * 2.0 ** -8) + grouped.abs().amax(-1) * 2.0 ** -7
    else:
        step = grouped.abs().amax(-1) / 7
        bound = step * (0.5 + 7 * 2.0 ** -8 + 2.0 ** -8)
    assert ((got.unflatten(1, (-1, group)) - grouped).abs() <= bound[..., None]).all()
    x = torch.randn(3, 5, k)
    want = x.double() @ got.double().T
    assert torch.allclose(lin(x).double(), want, atol=k * 2.0 ** -24 * float((x.abs() @ got.abs().T).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_input_of_a_4_bit_projection_gets_its_gradient(dtype):
    """g @ W, within the roundings of its type and of sums of 21 fp32 products; along a line the outputs change by it."""
    torch.manual_seed(2)
    lin = W.init_normal_(W.Int4Linear(96, 21), seed=3)
    w = hip.int4_dequantize(lin.weight, lin.scale, None, 21, 96).double()
    x = torch.randn(4, 96).to(dtype).requires_grad_()
    y = lin(x)
    g = torch.randn_like(y)
    y.backward(g)
    exact = g.double() @ w
    bound = 2.0 ** -8 * exact.abs() + 42 * 2.0 ** -24 * (g.double().abs() @ w.abs())
    assert x.grad.dtype == dtype and ((x.grad.double() - exact).abs() <= bound).all()
    if dtype is torch.float32:
        with torch.no_grad():
            d = torch.randn(4, 96)
            slope = ((lin(x + d) - lin(x - d)).double() * g.double()).sum() / 2
        sums = (x.detach().double().abs() + d.double().abs()) @ w.abs().T * g.double().abs()
        assert abs(slope - (x.grad.double() * d.double()).sum()) <= 2 * 96 * 2.0 ** -24 * sums.sum()


def test_what_a_4_bit_projection_refuses():
    with pytest.raises(ValueError, match="groups of 32"):
        W.Int4Linear(40, 16)
    with pytest.raises(ValueError, match="groups of 32"):
        W.Int4Linear(0, 16)
    with pytest.raises(ValueError, match="expected"):
        W.Int4Linear(64, 16).quantize_(torch.zeros(64, 16))
    lin = W.Int4Linear(64, 16)
    assert not lin.kernel_eligible(torch.zeros(2, 64, dtype=torch.bfloat16))  # on the host


def test_layer_bytes_are_those_of_the_parameters():
    for change in ({"int4": True}, {"int4": True, "qk_norm": True}, {"qk_norm": True}, {"int8": True, "qk_norm": True}, {}):
        shape = W.LlamaShape(n_layers=1, hidden=96, n_heads=2, n_kv_heads=1, head_dim=64, inter=160, vocab=9, max_seq=8,
                             **change)
        layer = W.build_llama(shape).layers[0]
        assert sum(p.numel() * p.element_size() for p in layer.parameters()) == shape.layer_bytes()


def test_more_channels_than_a_launch_tells_apart_are_refused():
    lib, b = nat.load(), ctypes.c_size_t(0)
    assert lib.ftx_int4_linear_workspace(1, 1 << 27, 128, 128, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert lib.ftx_int4_linear_workspace(1, 1 << 33, 128, 128, ctypes.byref(b)) == nat.FTX_ERR_UNSUPPORTED
