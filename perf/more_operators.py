"""The operators of a decoder that answers several tokens a pass, as measurable cases.

A pass of a streamed decoder costs its weights' bytes: 4-bit weights with a scale for each group of a channel's inputs
(``hip.int4_linear``) make them fewer, and a tree of drafted tokens that one pass checks makes more of them. The tree's
queries and keys are normalised for each head and turned by positions of their own on their way into the paged 8-bit
cache (``kv_cache.append``), attend over the cache and their ancestors (``kv_cache.tree_attention``), the accepted ones
move up behind the prefix in all layers (``kv_cache.keep``), and the logits of the nodes become log probabilities,
entropy and the likeliest tokens (``hip.token_logprobs``).

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass (the framework's where ``own`` is true, else the plain form in 32 bits),
``work`` what the pass cannot do without and ``exact`` the result in 64 bits.

A cache layer is ``codes`` [pages, 2, kv heads, blocks of a page, 32 d] (keys, then values) and ``scales`` [pages, 2,
kv heads, blocks of a page]. The 32 x d keys of a block are stored as [d / 16, 32, 16], its values as [d, 32].

A 4-bit weight [n, k] is ``weight`` [n / 16, k / 128, 1024] bytes (rounded up): the 16 bytes of lane 16 q + r hold, for
i < 4, the codes of channel r and inputs 32 i + 8 q + (0 .. 7) as a 32-bit word, input 2 j at bit 4 j and 2 j + 1 at bit
16 + 4 j. ``scale`` and ``zero`` are [n / 16, k / 128, 16, 128 / group].
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32  # tokens that share a scale
TINY = 2.0 ** -100  # a largest value whose scale is below this counts as zero
KINDS = {"fp8": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
LOGITS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5

# The decoder shapes of the benchmark, by the dimensions that these operators see.
_7B = {"heads": 32, "kv_heads": 32, "head_dim": 128}
_70B = {"heads": 64, "kv_heads": 8, "head_dim": 128}


def listed() -> list[dict]:
    return [
        # one token through an attention projection of the 7B decoder
        {"name": "int4_1_row", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False},
        # a small tree's nodes through the 70B decoder's gate projection
        {"name": "int4_13_rows", "kind": "linear", "m": 13, "n": 28672, "k": 8192, "group": 64, "zeros": True},
        # a prompt's rows, which fill no tile, through its down projection
        {"name": "int4_777_rows", "kind": "linear", "m": 777, "n": 8192, "k": 28672, "group": 128, "zeros": False},
        # the nodes of eight sequences' trees: several nodes of one position each
        {"name": "append_nodes_8x25", "kind": "append", **_70B, "codes": "fp8", "page": 64, "batch": 8, "new": 25,
         "ragged": False, "tree": True, "start": 4011},
        # a whole prompt into an empty cache, keys and queries normalised
        {"name": "append_prompt_2048", "kind": "append", **_7B, "codes": "int8", "page": 64, "batch": 1, "new": 2048,
         "ragged": False, "tree": False, "start": 0},
        # the smallest tree: one sequence's few nodes a little into its answer
        {"name": "tree_1x13_at_700", "kind": "tree", **_7B, "codes": "fp8", "page": 64, "batch": 1, "new": 13,
         "ragged": False, "start": 700},
        # a serving batch, trees of different sizes at different positions
        {"name": "tree_8x25_ragged_4096", "kind": "tree", **_70B, "codes": "int8", "page": 64, "batch": 8, "new": 25,
         "ragged": True, "start": 4096},
        # the largest trees over long contexts
        {"name": "tree_16x64_at_32000", "kind": "tree", **_70B, "codes": "fp8", "page": 128, "batch": 16, "new": 64,
         "ragged": False, "start": 32000},
        # one sequence's accepted path
        {"name": "keep_1x4", "kind": "keep", **_7B, "codes": "fp8", "page": 64, "layers": 32, "batch": 1, "nodes": 25,
         "kept": 4, "ragged": False, "start": 1003},
        # a batch's paths of different lengths in a deep model
        {"name": "keep_32x9", "kind": "keep", **_70B, "codes": "int8", "page": 64, "layers": 80, "batch": 32,
         "nodes": 64, "kept": 9, "ragged": True, "start": 321},
        # one decode token's logits
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 32000, "type": "fp32", "top": 5},
        # the log probabilities of a prompt
        {"name": "logprobs_2048", "kind": "logprobs", "rows": 2048, "vocab": 32000, "type": "bf16", "top": 20},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "append", "tree", "tree", "keep", "logprobs"])
    if kind == "linear":
        group = rng.choice([32, 64, 128])
        m = rng.choice([rng.randint(1, 16), _spread(rng, 17, 777)])
        return {"kind": kind, "m": m, "n": _spread(rng, 257, 28672), "group": group, "zeros": rng.random() < 0.5,
                "k": group * _spread(rng, 256 // group, 8192 // group)}
    if kind == "logprobs":
        vocab = _spread(rng, 1000, 131072)
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(2048, (1 << 26) // vocab))), "vocab": vocab,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "top": rng.choice([0, 1, rng.randint(2, 64)])}
    heads, kv, d = rng.choice([(32, 32, 128), (64, 8, 128), (16, 4, 64), (24, 8, 64), (12, 12, 128), (20, 4, 128)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv, "head_dim": d, "codes": rng.choice(["fp8", "int8"]),
         "page": rng.choice([32, 64, 128]), "ragged": rng.random() < 0.5}
    if kind == "keep":
        nodes = rng.randint(2, 64)
        return {**c, "layers": _spread(rng, 1, 640 // max(kv, 8)), "batch": _spread(rng, 1, 32), "nodes": nodes,
                "kept": rng.randint(1, min(nodes, 12)), "start": _spread(rng, 1, 321) - 1}
    if kind == "append":
        tree = rng.random() < 0.5
        new = rng.randint(1, 64) if tree else rng.choice([1, _spread(rng, 2, 1777)])
        batch = _spread(rng, 1, max(1, min(32, 1777 // new)))
        return {**c, "batch": batch, "new": new, "tree": tree, "start": _spread(rng, 1, 4096) - 1}
    batch = _spread(rng, 1, 16)
    return {**c, "batch": batch, "new": rng.randint(1, 64),
            "start": _spread(rng, 1, 32000 if batch * kv <= 128 else 8192)}


# ---- inputs -------------------------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) + 54321)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(*shape, device=DEV, generator=g)


def _uniform(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.rand(*shape, device=DEV, generator=g)


def _pool(case: dict, g: torch.Generator, *lead: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A pool of pages in use: codes as quantising normal values gives them, scales that differ by block."""
    dtype, top = KINDS[case["codes"]]
    shape = (*lead, 2, case["kv_heads"], case["page"] // BLOCK, BLOCK * case["head_dim"])
    codes = torch.empty(shape, dtype=dtype, device=DEV)
    for part in codes.view(torch.uint8).view(-1).split(1 << 27):  # the largest pool in 32 bits is no small tensor
        y = _normal(g, part.numel()).mul_(top / 4).clamp_(-top, top)
        part.copy_((y.round_() if dtype == torch.int8 else y).to(dtype).view(torch.uint8))
    scales = torch.exp(0.3 * _normal(g, *shape[:-1])) * (4 / top)
    return codes, scales


def _trees(g: torch.Generator, batch: int, nodes: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Random trees, parents before children: [batch, nodes] sets of ancestors (a bit each, the node's own included),
    and depths."""
    part = torch.rand(batch, nodes, device=DEV, generator=g).cpu()
    sets = torch.zeros(batch, nodes, dtype=torch.int64)
    depth = torch.zeros(batch, nodes, dtype=torch.int32)
    for i in range(nodes):
        bit = 1 << i if i < 63 else -(1 << 63)
        if i == 0:
            sets[:, 0] = bit
            continue
        # a parent among the nodes of the last half: deep rather than flat, as drafts are
        parent = (i // 2 + (part[:, i] * (i - i // 2)).long()).clamp(max=i - 1)[:, None]
        sets[:, i] = sets.gather(1, parent)[:, 0] | bit
        depth[:, i] = depth.gather(1, parent)[:, 0] + 1
    return sets.to(DEV), depth.to(DEV)


def _table(case: dict, g: torch.Generator, tokens: int) -> tuple[torch.Tensor, int]:
    width = -(-tokens // case["page"])
    pages = case["batch"] * width + 3
    order = torch.randperm(pages, device=DEV, generator=g)[: case["batch"] * width]
    return order.view(case["batch"], width).int(), pages


def _starts(case: dict, g: torch.Generator, most: int) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Cached tokens and new ones of each sequence; ragged: each its own, the first one the full ones."""
    b = case["batch"]
    if not case["ragged"]:
        return torch.full((b,), case["start"], dtype=torch.int32, device=DEV), None
    part = _uniform(g, 2, b)
    part[:, 0] = 1.0
    return (part[0] * case["start"]).floor().int(), (part[1] * (most + 1)).floor().clamp_(1, most).int()


def _rows(case: dict, seed: int) -> dict:
    """What append and the attention take."""
    g = _gen(seed)
    b, t, h, kv, d = case["batch"], case["new"], case["heads"], case["kv_heads"], case["head_dim"]
    starts, new = _starts(case, g, t)
    table, pages = _table(case, g, case["start"] + t)
    codes, scales = _pool(case, g, pages)
    s = {"codes": codes, "scales": scales, "table": table, "starts": starts, "new": new,
         "max_tokens": case["start"] + t, "q": _normal(g, b, t, h, d).bfloat16()}
    if case["kind"] == "tree":
        s["q"] *= 2.0  # scores some units apart: a few hundred keys of a long context have most of the weight
        s["tree"], _ = _trees(g, b, t)
        return s
    top = torch.ones(d, device=DEV)
    top[d // 8:: d // 4] = 4.0  # a few channels larger than the rest, as keys have them
    s["k"] = (_normal(g, b, t, kv, d) * top).bfloat16()
    s["v"] = _normal(g, b, t, kv, d).bfloat16()
    s["q_norm"], s["k_norm"] = ((1.0 + 0.2 * _normal(g, d)).bfloat16() for _ in range(2))
    s["positions"] = None
    if case["tree"]:
        s["positions"] = (starts[:, None] + _trees(g, b, t)[1]).int()
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
    ang = torch.outer(torch.arange(case["start"] + t, dtype=torch.float32), inv)
    ang = torch.cat([ang, ang], -1)
    s["cos"], s["sin"] = ang.cos().to(DEV), ang.sin().to(DEV)
    return s


def _keep_state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    table, pages = _table(case, g, case["start"] + case["nodes"])
    starts, counts = _starts(case, g, case["kept"])
    codes, scales = _pool(case, g, case["layers"], pages)
    # a path down the tree: the root, then nodes ever further on
    order = _uniform(g, case["batch"], case["nodes"])
    order[:, 0] = -1.0
    path = order.argsort(1)[:, : case["kept"]].sort(1).values.int()
    return {"codes": codes, "scales": scales, "table": table, "starts": starts, "path": path, "counts": counts}


def _linear_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    x = _normal(g, m, k)
    x[:, :: max(1, k // 8)] *= 8.0  # a few channels larger than the rest, as activations have them
    tiles, units = -(-n // 16), -(-k // 128)
    codes = torch.zeros(tiles * 16, units * 128, dtype=torch.uint8, device=DEV)
    codes[:n, :k] = _normal(g, n, k).mul_(2.8).add_(8.0).round_().clamp_(0, 15).byte()
    # [tile, channel, unit, i, q, j / 2, j % 2, half] -> bytes of [tile, unit, q, channel, i, half, j / 2], j % 2 = 0 in
    # the low bits
    c = codes.view(tiles, 16, units, 4, 4, 2, 2, 2).permute(0, 2, 4, 1, 3, 7, 5, 6)
    weight = (c[..., 0] | c[..., 1] << 4).reshape(tiles, units, 1024)
    shape = (tiles, units, 16, 128 // group)
    scale = (torch.exp(0.2 * _normal(g, *shape)) * (0.02 / 2.8)).bfloat16()
    zero = (8.0 + 1.5 * _normal(g, *shape)).round_().clamp_(0, 15).bfloat16() if case["zeros"] else None
    return {"x": x.bfloat16(), "weight": weight, "scale": scale, "zero": zero}


def _logprob_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    logits = _normal(g, rows, vocab).mul_(2.5)
    likely = torch.randint(0, vocab, (rows, 8), device=DEV, generator=g)
    logits.scatter_add_(1, likely, 6.0 + 2.0 * _normal(g, rows, 8))  # a few tokens stand out
    logits[:, vocab - vocab // 100:] = float("-inf")  # places of the table that are no tokens
    tokens = torch.where(_uniform(g, rows) < 0.7, likely[:, 0].clamp(max=vocab - vocab // 100 - 1),
                         torch.randint(0, vocab - vocab // 100, (rows,), device=DEV, generator=g))
    if rows > 8:
        tokens[:: 7] = -1  # padding: rows without a token
    return {"logits": logits.to(LOGITS[case["type"]]), "tokens": tokens}


@torch.no_grad()
def prepare(case: dict, seed: int) -> dict:
    make = {"linear": _linear_inputs, "keep": _keep_state, "logprobs": _logprob_inputs}.get(case["kind"], _rows)
    return {"case": dict(case), **make(case, seed)}


# ---- the plain form, in 32 bits -------------------------------------------------------------------------


def _to_codes(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    top = 127.0 if dtype == torch.int8 else 448.0
    y = y.clamp(-top, top)
    return torch.nan_to_num(y).round().to(dtype) if dtype == torch.int8 else y.to(dtype)


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin


def _block_values(codes: torch.Tensor, kv: int, d: int) -> torch.Tensor:
    """The codes of [..., 2, kv, 32 d] blocks as numbers, [..., 2, kv, 32, d]."""
    c = codes.float()
    keys = c[..., 0, :, :].unflatten(-1, (d // 16, BLOCK, 16)).transpose(-3, -2).flatten(-2)
    values = c[..., 1, :, :].unflatten(-1, (d, BLOCK)).transpose(-2, -1)
    return torch.stack((keys, values), -4)


def _block_codes(y: torch.Tensor, d: int) -> torch.Tensor:
    """[..., 2, kv, 32, d] bytes in the blocks' order, [..., 2, kv, 32 d]."""
    keys = y[..., 0, :, :, :].unflatten(-1, (d // 16, 16)).transpose(-3, -2).flatten(-3)
    values = y[..., 1, :, :, :].transpose(-2, -1).flatten(-2)
    return torch.stack((keys, values), -3)


def _normed(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """The factor in 64 bits: codes are the nearest ones to the results, some of which lie next to a border."""
    factor = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()
    return x.float() * factor * weight.float()


def _plain_append(s: dict):
    q, k, v = _normed(s["q"], s["q_norm"]), _normed(s["k"], s["k_norm"]), s["v"]
    b, t, kv, d = k.shape
    codes, scales, starts = s["codes"], s["scales"], s["starts"].long()
    new = s["new"].long() if s["new"] is not None else torch.full_like(starts, t)
    per_page = s["case"]["page"] // BLOCK
    i = torch.arange(t, device=DEV)
    at = s["positions"].long() if s["positions"] is not None else starts[:, None] + i
    at = at.clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at].unsqueeze(2), s["sin"][at].unsqueeze(2)
    live = i < new[:, None]
    q_out = torch.where(live[:, :, None, None], _rotate(q, cos, sin), 0.0).bfloat16()
    fresh = torch.stack((_rotate(k, cos, sin), v.float()), 2)  # [b, t, 2, kv, d]

    first = starts // BLOCK
    blocks = (t + BLOCK - 1) // BLOCK + 1  # the most that t tokens touch
    block = first[:, None] + torch.arange(blocks, device=DEV)
    written = block * BLOCK < (starts + new)[:, None]
    page = s["table"].long().gather(1, (block // per_page).clamp(max=s["table"].shape[1] - 1))
    seq, nth = written.nonzero(as_tuple=True)
    page, part = page[seq, nth], (block % per_page)[seq, nth]
    token = block[seq, nth][:, None] * BLOCK + torch.arange(BLOCK, device=DEV) - starts[seq][:, None]
    is_new = (token >= 0) & (token < new[seq][:, None])  # [touched blocks, 32]
    is_old = token < 0
    y = fresh[seq[:, None], token.clamp(0, t - 1)].permute(0, 2, 3, 1, 4)  # [touched, 2, kv, 32, d]
    of = is_new[:, None, None, :, None]
    top = 127.0 if codes.dtype == torch.int8 else 448.0
    largest = torch.where(of & y.isfinite(), y.abs(), 0.0).amax((-2, -1))
    mine = codes.view(torch.uint8)
    old_codes = mine[page, :, :, part].view(codes.dtype)
    old_scale = torch.where(is_old[:, :1, None], scales[page, :, :, part], 0.0)
    made = largest * torch.tensor(1.0 / top, dtype=torch.float32)
    scale = torch.maximum(old_scale, torch.where(made < TINY, 0.0, made))
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    old = _block_values(old_codes, kv, d)
    ratio = torch.where(scale > old_scale, old_scale * inverse, 1.0)
    value = torch.where(of, y * inverse[..., None, None], old * ratio[..., None, None])
    value = torch.where((is_new | is_old)[:, None, None, :, None], value, 0.0)
    mine[page, :, :, part] = _block_codes(_to_codes(value, codes.dtype).view(torch.uint8), d)
    scales[page, :, :, part] = scale
    return q_out


def _plain_tree(s: dict) -> torch.Tensor:
    q, case = s["q"], s["case"]
    b, t, h, d = q.shape
    kv = case["kv_heads"]
    starts = s["starts"].long()
    new = s["new"].long() if s["new"] is not None else torch.full_like(starts, t)
    table = s["table"].long()
    cached = s["codes"].view(torch.uint8)[table].view(s["codes"].dtype)  # [b, width, 2, kv, blocks, 32 d]
    cached = _block_values(cached.permute(0, 1, 4, 2, 3, 5).flatten(1, 2), kv, d)
    factor = s["scales"][table].permute(0, 1, 4, 2, 3).flatten(1, 2)  # [b, blocks, 2, kv]
    cached = (cached * factor[..., None, None]).permute(2, 0, 3, 1, 4, 5).flatten(3, 4)  # [2, b, kv, tokens, d]
    keys, values = cached[0], cached[1]
    p = torch.arange(keys.shape[2], device=DEV)
    values = values.masked_fill((p >= (starts + t)[:, None])[:, None, :, None], 0.0)
    rows = q.float().unflatten(2, (kv, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, t rep, d]
    scores = torch.matmul(rows, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    node = p - starts[:, None]  # [b, tokens]
    bit = (s["tree"][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    seen = (node < 0)[:, None] | ((bit != 0) & (node < t)[:, None])  # [b, t, tokens]
    seen = seen & (torch.arange(t, device=DEV) < new[:, None])[:, :, None]
    seen = seen.repeat_interleave(h // kv, 1)[:, None]
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = torch.exp(scores.sub_(top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values.contiguous()) / torch.where(total > 0, total, 1.0)
    return out.unflatten(2, (t, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous().bfloat16()


def _plain_keep(s: dict) -> None:
    """The blocks of the prefix's end and of the nodes, at most four a sequence, gathered, changed and put back."""
    codes, scales, case = s["codes"], s["scales"], s["case"]
    kv, d, per_page, kept = case["kv_heads"], case["head_dim"], case["page"] // BLOCK, case["kept"]
    starts, path = s["starts"].long(), s["path"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(starts, kept)
    held = (case["nodes"] + BLOCK - 2) // BLOCK + 1  # blocks that the nodes reach into
    block = (starts // BLOCK)[:, None] + torch.arange(held, device=DEV)
    page = s["table"].long().gather(1, (block // per_page).clamp(max=s["table"].shape[1] - 1))
    part = block % per_page
    mine = codes.view(torch.uint8)
    old_codes = mine[:, page, :, :, part].view(codes.dtype)  # [batch, blocks, layers, 2, kv, 32 d]
    old_scale = scales[:, page, :, :, part]  # [batch, blocks, layers, 2, kv]
    values = _block_values(old_codes, kv, d).movedim(-2, 2).flatten(1, 2)  # [batch, tokens, layers, 2, kv, d]
    token = torch.arange(held * BLOCK, device=DEV)
    start = (starts % BLOCK)[:, None]
    nth = token - start  # of the kept ones
    is_new = (nth >= 0) & (nth < counts[:, None])
    is_old = nth < 0
    source = torch.where(is_new, start + path.gather(1, nth.clamp(0, kept - 1)), token)  # [batch, tokens]
    at = torch.arange(case["batch"], device=DEV)[:, None]
    from_scale = old_scale[at, source // BLOCK]  # [batch, tokens, layers, 2, kv]
    used = (is_new | is_old)[:, :, None, None, None]
    scale = torch.where(used, from_scale, 0.0).unflatten(1, (held, BLOCK)).amax(2)
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0).repeat_interleave(BLOCK, 1)
    ratio = torch.where(scale.repeat_interleave(BLOCK, 1) > from_scale, from_scale * inverse, 1.0)
    value = torch.where(used[..., None], values[at, source] * ratio[..., None], 0.0)
    value = value.unflatten(1, (held, BLOCK)).movedim(2, -2)
    made = _block_codes(_to_codes(value, codes.dtype).view(torch.uint8), d)
    seq, which = (is_new.unflatten(1, (held, BLOCK)).any(-1)).nonzero(as_tuple=True)  # blocks that tokens move to
    mine[:, page[seq, which], :, :, part[seq, which]] = made[seq, which]
    scales[:, page[seq, which], :, :, part[seq, which]] = scale[seq, which]


def _plain_linear(s: dict) -> torch.Tensor:
    case = s["case"]
    tiles, units, _ = s["weight"].shape
    c = torch.stack((s["weight"] & 15, s["weight"] >> 4), -1).view(tiles, units, 4, 16, 4, 2, 2, 2)
    # [tile, unit, q, channel, i, half, j / 2, j % 2] -> [tile, channel, unit, i, q, j, half]
    c = c.permute(0, 3, 1, 4, 2, 6, 7, 5).reshape(tiles * 16, units * (128 // case["group"]), case["group"]).float()
    scale = s["scale"].float().transpose(1, 2).reshape(tiles * 16, -1, 1)
    zero = s["zero"].float().transpose(1, 2).reshape(tiles * 16, -1, 1) if s["zero"] is not None else 8.0
    w = ((c - zero) * scale).flatten(1)[: case["n"], : case["k"]]
    return torch.matmul(s["x"].float(), w.t()).bfloat16()


def _plain_logprobs(s: dict):
    x, tokens, top = s["logits"].float(), s["tokens"], s["case"]["top"]
    vocab = x.shape[1]
    most = x.amax(-1, keepdim=True)
    shifted = x - most
    weight = torch.exp(shifted)
    total = weight.sum(-1, keepdim=True)
    log_total = torch.log(total)
    given = shifted.gather(1, tokens.clamp(0, vocab - 1)[:, None]) - log_total
    given = torch.where(tokens >= 0, given[:, 0], 0.0)
    part = torch.where(weight > 0, shifted * weight, 0.0).sum(-1, keepdim=True)
    entropy = (log_total - part / total)[:, 0]
    # whole numbers in the order of the logits, equal ones by their index, lowest first
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    index = (bits * (1 << 24) + (vocab - 1 - torch.arange(vocab, device=DEV))).topk(top, -1).indices
    return given, entropy, shifted.gather(1, index) - log_total, index


@torch.no_grad()
def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        from flextensor_amd import hip, kv_cache

        if kind == "linear":
            return hip.int4_linear(s["x"], s["weight"], s["scale"], s["zero"], n=s["case"]["n"])
        if kind == "logprobs":
            return hip.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
        if kind == "tree":
            return kv_cache.tree_attention(s["q"], s["codes"], s["scales"], s["table"], s["starts"], s["tree"],
                                           s["new"], max_tokens=s["max_tokens"])
        if kind == "keep":
            kv_cache.keep(s["codes"], s["scales"], s["table"], s["starts"], s["path"], s["counts"])
            return {"codes": s["codes"], "scales": s["scales"]}
        q = kv_cache.append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["codes"], s["scales"], s["table"],
                            s["starts"], s["new"], positions=s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                            eps=EPS)
        return {"q": q, "codes": s["codes"], "scales": s["scales"]}
    if kind == "linear":
        return _plain_linear(s)
    if kind == "logprobs":
        return _plain_logprobs(s)
    if kind == "tree":
        return _plain_tree(s)
    if kind == "keep":
        _plain_keep(s)
        return {"codes": s["codes"], "scales": s["scales"]}
    # The codes are what the cache holds: both forms round the same 32-bit values, so they are the same codes.
    return {"q": _plain_append(s), "codes": s["codes"], "scales": s["scales"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        part = (4 if case["zeros"] else 2) / case["group"]
        return {"bytes": float(n * k * (0.5 + part) + 2 * m * k + 2 * m * n), "flops": 2.0 * m * n * k}
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": float(rows * (vocab * LOGITS[case["type"]].itemsize + 8 + 8 + 12 * case["top"])),
                "flops": 4.0 * rows * vocab}
    kv, d = case["kv_heads"], case["head_dim"]
    token = 2 * kv * (d + 4 / BLOCK)  # a cached token's codes and its part of the scales
    b, start = case["batch"], case["start"]
    if kind == "keep":
        # Values lie a block of 32 tokens together: what a path names is read, and what it moves to written, by blocks.
        kept = case["kept"] if not case["ragged"] else (case["kept"] + 1) / 2
        read = min(1 + (case["nodes"] - 1) / BLOCK, kept)
        return {"bytes": float(case["layers"] * b * BLOCK * token * (read + 1 + (kept - 1) / BLOCK)), "flops": 0.0}
    h, t = case["heads"], case["new"]
    if case["ragged"]:  # the first sequence has it all, the others half on average
        new, before = t + (b - 1) * (t + 1) / 2, start * (1 + (b - 1) / 2)
    else:
        new, before = b * t, b * start
    if kind == "append":
        return {"bytes": float(new * (4 * h * d + 4 * kv * d + token)), "flops": float(new * (h + kv) * 7 * d)}
    pairs = new * (before / b + 4)  # a node sees the prefix and some ancestors
    return {"bytes": float((before + b * t) * token + 4 * new * h * d), "flops": float(4 * h * d * pairs)}


# ---- the same results in 64 bits ----------------------------------------------------------------------------


def _round64(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The nearest number that an 8-bit code stands for, ties to even."""
    if dtype == torch.int8:
        return y.round()
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)  # three bits after the leading one, 2^-9 between subnormals
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def _cells(block: torch.Tensor, side: int, d: int) -> torch.Tensor:
    """[..., 32 d] codes of one side's block as [..., 32, d]."""
    if side == 0:
        return block.unflatten(-1, (d // 16, BLOCK, 16)).transpose(-3, -2).flatten(-2)
    return block.unflatten(-1, (d, BLOCK)).transpose(-2, -1)


def _from_cells(cells: torch.Tensor, side: int, d: int) -> torch.Tensor:
    if side == 0:
        return cells.unflatten(-1, (d // 16, 16)).transpose(-3, -2).flatten(-3)
    return cells.transpose(-2, -1).flatten(-2)


def _exact_append(case: dict, seed: int) -> dict:
    """Sequence by sequence and block by block, on the tokens' own [32, d] values."""
    s = _rows(case, seed)
    codes, scales = s["codes"], s["scales"].double()
    b, t, kv, d = s["k"].shape
    top = 127.0 if codes.dtype == torch.int8 else 448.0
    half, page_tokens = d // 2, case["page"]
    held = codes.double()
    counts = [t] * b if s["new"] is None else s["new"].tolist()
    q_out = torch.zeros_like(s["q"], dtype=torch.float64)
    table = s["table"].tolist()

    def ready(x, weight, cos, sin):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        lo, hi = x[..., :half], x[..., half:]
        return torch.cat((lo * cos[..., :half] - hi * sin[..., :half], hi * cos[..., half:] + lo * sin[..., half:]), -1)

    for n, start in enumerate(s["starts"].tolist()):
        count = counts[n]
        at = torch.arange(start, start + count, device=DEV)
        if s["positions"] is not None:
            at = s["positions"][n, :count].long()
        cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
        q_out[n, :count] = ready(s["q"][n, :count], s["q_norm"], cos, sin)
        pair = (ready(s["k"][n, :count], s["k_norm"], cos, sin), s["v"][n, :count].double())
        for block in range(start // BLOCK, (start + count - 1) // BLOCK + 1):
            page, part = table[n][block * BLOCK // page_tokens], block % (page_tokens // BLOCK)
            lo, hi = max(start, block * BLOCK), min(start + count, (block + 1) * BLOCK)
            for side in range(2):
                rows = pair[side][lo - start: hi - start].transpose(0, 1)  # [kv, tokens, d]
                before = lo - block * BLOCK  # tokens of earlier calls
                was = scales[page, side, :, part] if before else torch.zeros(kv, dtype=torch.float64, device=DEV)
                now = torch.maximum(was, rows.abs().amax((1, 2)) / top)
                safe = torch.where(now > 0, now, 1.0)
                cells = _cells(held[page, side, :, part], side, d).clone()
                older = cells[:, :before] * (was / safe)[:, None, None]
                grown = (now > was)[:, None, None]
                cells[:, :before] = torch.where(grown, _round64(older, codes.dtype), cells[:, :before])
                cells[:, before: before + hi - lo] = _round64(rows / safe[:, None, None], codes.dtype)
                cells[:, before + hi - lo:] = 0.0
                held[page, side, :, part] = _from_cells(cells, side, d)
                scales[page, side, :, part] = now
    return {"q": q_out, "codes": held if codes.dtype != torch.int8 else None, "scales": scales}


def _exact_tree(case: dict, seed: int) -> torch.Tensor:
    """Sequence by sequence and head by head, the keys a sequence has and no others."""
    s = _rows(case, seed)
    b, t, h, d = s["q"].shape
    kv, rep = case["kv_heads"], h // case["kv_heads"]
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=DEV)
    counts = [t] * b if s["new"] is None else s["new"].tolist()
    raw = s["codes"].view(torch.uint8)
    for n, start in enumerate(s["starts"].tolist()):
        length = start + t
        pages = s["table"][n, : -(-length // case["page"])].long()
        sets = [v & (2 ** 64 - 1) for v in s["tree"][n, : counts[n]].tolist()]
        seen = torch.ones(counts[n], length, dtype=torch.bool)
        seen[:, start:] = torch.tensor([[v >> j & 1 for j in range(t)] for v in sets], dtype=torch.bool)
        seen = seen.to(DEV).repeat_interleave(rep, 0)
        for j in range(kv):
            c = raw[pages, :, j].view(s["codes"].dtype).double() * s["scales"][pages, :, j].double()[..., None]
            keys = _cells(c[:, 0], 0, d).reshape(-1, d)[:length]
            values = _cells(c[:, 1], 1, d).reshape(-1, d)[:length]
            rows = s["q"][n, : counts[n], j * rep: (j + 1) * rep].double()
            scores = rows.flatten(0, 1) @ keys.t().contiguous() / math.sqrt(d)
            mixed = torch.softmax(scores.masked_fill(~seen, float("-inf")), -1) @ values.contiguous()
            out[n, : counts[n], j * rep: (j + 1) * rep] = mixed.unflatten(0, (counts[n], rep))
    return out


def _exact_keep(case: dict, seed: int) -> dict:
    """Token by token: the numbers that the accepted nodes stand for, then the blocks that they move to."""
    s = _keep_state(case, seed)
    codes, scales = s["codes"], s["scales"].double()
    raw = codes.view(torch.uint8)
    d, page_tokens = case["head_dim"], case["page"]
    table, paths = s["table"].tolist(), s["path"].tolist()
    counts = [case["kept"]] * case["batch"] if s["counts"] is None else s["counts"].tolist()
    written = {}
    for n, start in enumerate(s["starts"].tolist()):
        places = [start + p for p in paths[n][: counts[n]]]
        for block in range(start // BLOCK, (start + counts[n] - 1) // BLOCK + 1):
            tokens = [p if p < start else places[p - start]
                      for p in range(block * BLOCK, min((block + 1) * BLOCK, start + counts[n]))]
            where = [(table[n][p // page_tokens], p // BLOCK % (page_tokens // BLOCK), p % BLOCK) for p in tokens]
            was = torch.stack([scales[:, page, :, :, part] for page, part, _ in where], -1)  # [layers, 2, kv, tokens]
            now = was.amax(-1)
            sides = []
            for side in range(2):
                cells = torch.zeros(*now.shape[:1], now.shape[2], BLOCK, d, dtype=torch.float64, device=DEV)
                for i, (page, part, token) in enumerate(where):
                    cell = _cells(raw[:, page, side, :, part].view(codes.dtype).double(), side, d)[:, :, token]
                    ratio = (was[:, side, :, i] / now[:, side])[..., None]
                    cells[:, :, i] = torch.where(ratio < 1, _round64(cell * ratio, codes.dtype), cell)
                sides.append(_from_cells(cells, side, d))
            written[table[n][block * BLOCK // page_tokens], block % (page_tokens // BLOCK)] = (sides, now)
    held = codes.double()
    for (page, part), (sides, now) in written.items():
        held[:, page, 0, :, part], held[:, page, 1, :, part] = sides
        scales[:, page, :, :, part] = now
    return {"codes": held if codes.dtype != torch.int8 else None, "scales": scales}


def _exact_linear(case: dict, seed: int) -> torch.Tensor:
    """Tile by tile of 16 channels, input by input of a word."""
    s = _linear_inputs(case, seed)
    n, k, group = case["n"], case["k"], case["group"]
    tiles, units, _ = s["weight"].shape
    words = s["weight"].view(torch.int32).view(tiles, units, 4, 16, 4)  # [tile, unit, q, channel, i]
    y = torch.empty(case["m"], tiles * 16, dtype=torch.float64, device=DEV)
    x = torch.zeros(case["m"], units * 128, dtype=torch.float64, device=DEV)
    x[:, :k] = s["x"].double()
    of_group = torch.arange(128, device=DEV) // group
    for first in range(0, tiles, 64):
        part = words[first: first + 64]
        w = torch.empty(part.shape[0], 16, units, 128, dtype=torch.float64, device=DEV)
        for i in range(4):
            for q in range(4):
                for e in range(8):
                    c = (part[:, :, q, :, i] >> (4 * (e // 2) + 16 * (e % 2))) & 15
                    w[..., 32 * i + 8 * q + e] = c.transpose(1, 2).double()
        scale, zero = (p[first: first + 64].double().transpose(1, 2)[..., of_group] if p is not None else 8.0
                       for p in (s["scale"], s["zero"]))
        y[:, first * 16: first * 16 + part.shape[0] * 16] = x @ ((w - zero) * scale).view(-1, units * 128).t()
    return y[:, :n]


def _exact_logprobs(case: dict, seed: int):
    s = _logprob_inputs(case, seed)
    given, entropy, best, index = [], [], [], []
    for x, tokens in zip(s["logits"].split(256), s["tokens"].split(256)):
        logp = torch.log_softmax(x.double(), -1)
        given.append(torch.where(tokens >= 0, logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0))
        entropy.append(-(logp.exp() * logp.masked_fill(logp == float("-inf"), 0.0)).sum(-1))
        order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, : case["top"]]
        best.append(logp.gather(1, order))
        index.append(order)
    return tuple(torch.cat(v) for v in (given, entropy, best, index))


@torch.no_grad()
def exact(case: dict, seed: int):
    make = {"append": _exact_append, "tree": _exact_tree, "keep": _exact_keep, "linear": _exact_linear,
            "logprobs": _exact_logprobs}[case["kind"]]
    return make(case, seed)
