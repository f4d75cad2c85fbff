"""The operators of serving in 8 bits, as measurable cases.

A KV cache held in pages of 8-bit codes, with a scale for each 32 tokens of a head: writing new positions into it
(``kv_cache.append``), attention over it (``kv_cache.attention``) and copying its pages when a sequence is forked or
the pool compacted (``kv_cache.copy_pages``); and the matrix product of 8-bit integers with a scale for each token
and each channel (``hip.int8_linear``).

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass (the framework's where ``own`` is true, else the plain form in 32 bits),
``work`` what the pass cannot do without and ``exact`` the result in 64 bits.

A cache layer is ``codes`` [pages, 2, kv heads, blocks of a page, 32 d] (keys, then values) and ``scales`` [pages, 2,
kv heads, blocks of a page]. The 32 x d keys of a block are stored as [d / 16, 32, 16], its values as [d, 32].
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32  # tokens that share a scale
TINY = 2.0 ** -100  # a largest value whose scale is below this counts as zero
KINDS = {"fp8": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}

# The decoder shapes of the benchmark, by the dimensions that these operators see.
_7B = {"heads": 32, "kv_heads": 32, "head_dim": 128}
_70B = {"heads": 64, "kv_heads": 8, "head_dim": 128}


def listed() -> list[dict]:
    return [
        # a decode step of eight sequences: one new token each, somewhere in a block that holds others
        {"name": "append_decode_8", "kind": "append", **_70B, "codes": "fp8", "page": 64, "batch": 8, "new": 1,
         "ragged": False, "start": 4011},
        # a whole prompt into an empty cache
        {"name": "append_prompt_2048", "kind": "append", **_7B, "codes": "int8", "page": 64, "batch": 1, "new": 2048,
         "ragged": False, "start": 0},
        # prompts of different lengths that continue cached prefixes, in a small model's heads
        {"name": "append_ragged_777", "kind": "append", "heads": 16, "kv_heads": 4, "head_dim": 64, "codes": "fp8",
         "page": 32, "batch": 5, "new": 777, "ragged": True, "start": 1000},
        # the smallest attention: one sequence's token a little into its answer
        {"name": "attend_1_at_100", "kind": "attend", **_7B, "codes": "fp8", "page": 64, "batch": 1, "new": 1,
         "ragged": False, "start": 100},
        # a serving batch of decode tokens at different positions
        {"name": "attend_8_ragged_4096", "kind": "attend", **_7B, "codes": "int8", "page": 64, "batch": 8, "new": 1,
         "ragged": True, "start": 4096},
        # decode over long contexts
        {"name": "attend_16_at_32000", "kind": "attend", **_70B, "codes": "fp8", "page": 128, "batch": 16, "new": 1,
         "ragged": False, "start": 32000},
        # a chunk of a long prompt over what came before it
        {"name": "attend_chunk_2048_at_6100", "kind": "attend", **_70B, "codes": "int8", "page": 64, "batch": 1,
         "new": 2048, "ragged": False, "start": 6100},
        # forking a sequence inside its last page: that page's copy in every layer
        {"name": "copy_fork", "kind": "copy", **_7B, "codes": "fp8", "page": 64, "layers": 32, "pool": 24, "moved": 1},
        # compaction: the pages in use at the pool's end move to the free ones at its start
        {"name": "copy_compact_40", "kind": "copy", **_70B, "codes": "int8", "page": 64, "layers": 80, "pool": 97,
         "moved": 40},
        # one token through an attention projection of the 7B decoder
        {"name": "linear_1_row", "kind": "linear", "m": 1, "n": 4096, "k": 4096},
        # a decode batch of odd size through the 70B decoder's gate projection
        {"name": "linear_13_rows", "kind": "linear", "m": 13, "n": 28672, "k": 8192},
        # a prompt's rows, which fill no tile, through the same projection
        {"name": "linear_2111_rows", "kind": "linear", "m": 2111, "n": 28672, "k": 8192},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "attend", "copy", "linear"])
    if kind == "linear":
        m = _spread(rng, 1, 2111)
        return {"kind": kind, "m": m, "n": _spread(rng, 257, 28672), "k": 16 * _spread(rng, 17, 512)}
    heads, kv, d = rng.choice([(32, 32, 128), (64, 8, 128), (16, 4, 64), (24, 8, 64), (12, 12, 128), (20, 4, 128)])
    c = {"kind": kind, "heads": heads, "kv_heads": kv, "head_dim": d, "codes": rng.choice(["fp8", "int8"]),
         "page": rng.choice([32, 64, 128])}
    if kind == "copy":
        moved = _spread(rng, 1, 40)
        return {**c, "layers": _spread(rng, 1, 24), "pool": 2 * moved + rng.randint(1, 9), "moved": moved}
    if kind == "append":
        new = rng.choice([1, _spread(rng, 2, 2048)])
        batch = _spread(rng, 1, 64 if new == 1 else max(1, min(8, 2048 // new)))
        return {**c, "batch": batch, "new": new, "ragged": rng.random() < 0.5, "start": _spread(rng, 1, 4096) - 1}
    if rng.random() < 0.6:  # decode, or a few tokens a sequence
        batch = _spread(rng, 1, 16)
        return {**c, "batch": batch, "new": rng.choice([1, 1, rng.randint(2, 7)]), "ragged": rng.random() < 0.5,
                "start": _spread(rng, 1, 32000 if batch * kv <= 128 else 8192)}
    new = _spread(rng, 8, 2048)
    return {**c, "batch": _spread(rng, 1, max(1, min(4, 2048 // new))), "new": new, "ragged": rng.random() < 0.5,
            "start": _spread(rng, 1, 6101) - 1}


# ---- inputs -------------------------------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) + 12345)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(*shape, device=DEV, generator=g)


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


def _state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    b, t, h, kv, d = case["batch"], case["new"], case["heads"], case["kv_heads"], case["head_dim"]
    if case["ragged"]:  # every sequence a start and a number of tokens of its own, the first one the full ones
        part = torch.rand(2, b, device=DEV, generator=g)
        part[:, 0] = 1.0
        starts = (part[0] * case["start"]).floor().int()
        new = (part[1] * (t + 1)).floor().clamp_(1, t).int()
    else:
        starts = torch.full((b,), case["start"], dtype=torch.int32, device=DEV)
        new = None
    width = -(-(case["start"] + t) // case["page"])
    pages = b * width + 3
    table = torch.randperm(pages, device=DEV, generator=g)[: b * width].view(b, width).int()
    codes, scales = _pool(case, g, pages)
    top = torch.ones(d, device=DEV)
    top[d // 8:: d // 4] = 4.0  # a few channels larger than the rest, as keys have them
    state = {"codes": codes, "scales": scales, "table": table, "starts": starts, "new": new,
             "max_tokens": case["start"] + t, "q": (_normal(g, b, t, h, d)).bfloat16()}
    if case["kind"] == "append":
        state["k"] = (_normal(g, b, t, kv, d) * top).bfloat16()
        state["v"] = _normal(g, b, t, kv, d).bfloat16()
        state["cos"], state["sin"] = _tables(d, case["start"] + t, torch.float32)
    else:
        state["q"] *= 2.0  # scores some units apart: a few hundred keys of a long context have most of the weight
    return state


def _tables(d: int, positions: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin of the rotary angles, in the precision that a model keeps them in."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
    ang = torch.outer(torch.arange(positions, dtype=torch.float32), inv)
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(DEV, dtype), ang.sin().to(DEV, dtype)


def _linear_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    m, n, k = case["m"], case["n"], case["k"]
    x = _normal(g, m, k)
    x[:, :: max(1, k // 8)] *= 8.0  # a few channels larger than the rest, as activations have them
    w = torch.empty(n, k, dtype=torch.int8, device=DEV)
    w.copy_(_normal(g, n, k).mul_(32.0).round_().clamp_(-127, 127))
    scale = torch.exp(0.2 * _normal(g, n)) * (0.02 / 32)
    return {"x": x.bfloat16(), "w": w, "scale": scale}


def _copy_state(case: dict, seed: int) -> dict:
    g = _gen(seed)
    codes, scales = _pool(case, g, case["layers"], case["pool"])
    order = torch.randperm(case["pool"] - case["moved"], device=DEV, generator=g)[: case["moved"]]
    dst = sorted(order.tolist())
    src = list(range(case["pool"] - case["moved"], case["pool"]))
    return {"codes": codes, "scales": scales, "src": src, "dst": dst,
            "src_index": torch.tensor(src, device=DEV), "dst_index": torch.tensor(dst, device=DEV)}


@torch.no_grad()
def prepare(case: dict, seed: int) -> dict:
    make = {"linear": _linear_inputs, "copy": _copy_state}.get(case["kind"], _state)
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


def _plain_append(s: dict):
    q, k, v = s["q"], s["k"], s["v"]
    b, t, kv, d = k.shape
    codes, scales, starts = s["codes"], s["scales"], s["starts"].long()
    new = s["new"].long() if s["new"] is not None else torch.full_like(starts, t)
    per_page = s["case"]["page"] // BLOCK
    i = torch.arange(t, device=DEV)
    at = (starts[:, None] + i).clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at].unsqueeze(2), s["sin"][at].unsqueeze(2)
    live = i < new[:, None]
    q_out = torch.where(live[:, :, None, None], _rotate(q.float(), cos, sin), 0.0).bfloat16()
    fresh = torch.stack((_rotate(k.float(), cos, sin), v.float()), 2)  # [b, t, 2, kv, d]

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


def _plain_attend(s: dict) -> torch.Tensor:
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
    values = values.masked_fill((p >= (starts + new)[:, None])[:, None, :, None], 0.0)
    rows = q.float().unflatten(2, (kv, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, t rep, d]
    scores = torch.matmul(rows, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    i = torch.arange(t, device=DEV)
    seen = (p <= (starts[:, None] + i)[:, :, None]) & (i < new[:, None])[:, :, None]  # [b, t, tokens]
    seen = seen.repeat_interleave(h // kv, 1)[:, None]
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = torch.exp(scores.sub_(top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values.contiguous()) / torch.where(total > 0, total, 1.0)
    return out.unflatten(2, (t, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous().bfloat16()


def _plain_linear(s: dict) -> torch.Tensor:
    x = s["x"].float()
    largest = x.abs().amax(-1, keepdim=True)
    made = largest * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    scale = torch.where(made < TINY, 0.0, made)
    codes = (x * torch.where(scale > 0, 1.0 / scale, 0.0)).round().clamp(-127, 127)
    return (torch.matmul(codes, s["w"].float().t()) * scale * s["scale"]).bfloat16()


@torch.no_grad()
def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        from flextensor_amd import hip, kv_cache

        if kind == "linear":
            return hip.int8_linear(s["x"], s["w"], s["scale"])
        if kind == "attend":
            return kv_cache.attention(s["q"], s["codes"], s["scales"], s["table"], s["starts"], s["new"],
                                      max_tokens=s["max_tokens"])
        if kind == "copy":
            kv_cache.copy_pages(s["codes"], s["scales"], s["src"], s["dst"])
            return {"codes": s["codes"], "scales": s["scales"]}
        q = kv_cache.append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["codes"], s["scales"], s["table"],
                            s["starts"], s["new"])
        return {"q": q, "codes": s["codes"], "scales": s["scales"]}
    if kind == "linear":
        return _plain_linear(s)
    if kind == "attend":
        return _plain_attend(s)
    if kind == "copy":
        codes = s["codes"].view(torch.uint8)
        codes[:, s["dst_index"]] = codes[:, s["src_index"]]
        s["scales"][:, s["dst_index"]] = s["scales"][:, s["src_index"]]
        return {"codes": s["codes"], "scales": s["scales"]}
    # The codes are what the cache holds: both forms round the same 32-bit values, so they are the same codes.
    return {"q": _plain_append(s), "codes": s["codes"], "scales": s["scales"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(n * k + 2 * m * k + 2 * m * n + 4 * n), "flops": 2.0 * m * n * k}
    kv, d = case["kv_heads"], case["head_dim"]
    token = 2 * kv * (d + 4 / BLOCK)  # a cached token's codes and its part of the scales
    if kind == "copy":
        return {"bytes": 2.0 * case["layers"] * case["moved"] * case["page"] * token, "flops": 0.0}
    h, b, t, start = case["heads"], case["batch"], case["new"], case["start"]
    if case["ragged"]:  # the first sequence has it all, the others half on average
        new, before = t + (b - 1) * (t + 1) / 2, start * (1 + (b - 1) / 2)
    else:
        new, before = b * t, b * start
    if kind == "append":
        return {"bytes": float(new * (4 * h * d + 4 * kv * d + token)), "flops": float(new * (h + kv) * 3 * d)}
    pairs = new * (before / b + (t + 1) / 2)  # the causal part of the new tokens' own
    return {"bytes": float((before + new) * token + 4 * new * h * d), "flops": float(4 * h * d * pairs)}


# ---- the same results in 64 bits ----------------------------------------------------------------------------


def _exact_append(case: dict, seed: int) -> dict:
    """Sequence by sequence and block by block, on the tokens' own [32, d] values."""
    s = _state(case, seed)
    k, v, codes, scales = s["k"].double(), s["v"].double(), s["codes"], s["scales"].double()
    b, t, kv, d = k.shape
    top = 127.0 if codes.dtype == torch.int8 else 448.0
    half, page_tokens = d // 2, case["page"]
    held = codes.double()
    counts = [t] * b if s["new"] is None else s["new"].tolist()
    q_out = torch.zeros_like(s["q"], dtype=torch.float64)
    table = s["table"].tolist()
    for n, start in enumerate(s["starts"].tolist()):
        count = counts[n]
        cos, sin = s["cos"][start: start + count].double(), s["sin"][start: start + count].double()

        def turn(x):
            lo, hi = x[..., :half], x[..., half:]
            c, z = cos[:, None], sin[:, None]
            return torch.cat((lo * c[..., :half] - hi * z[..., :half], hi * c[..., half:] + lo * z[..., half:]), -1)

        q_out[n, :count] = turn(s["q"][n, :count].double())
        pair = (turn(k[n, :count]), v[n, :count])
        for block in range(start // BLOCK, (start + count - 1) // BLOCK + 1):
            at, part = table[n][block * BLOCK // page_tokens], block % (page_tokens // BLOCK)
            lo = max(start, block * BLOCK)
            hi = min(start + count, (block + 1) * BLOCK)
            for side in range(2):
                rows = pair[side][lo - start: hi - start].transpose(0, 1)  # [kv, tokens, d]
                before = lo - block * BLOCK  # tokens of earlier calls
                was = scales[at, side, :, part] if before else torch.zeros(kv, dtype=torch.float64, device=DEV)
                now = torch.maximum(was, rows.abs().amax((1, 2)) / top)
                now_safe = torch.where(now > 0, now, 1.0)
                cells = held[at, side, :, part]
                cells = (cells.view(kv, d // 16, BLOCK, 16).transpose(1, 2).reshape(kv, BLOCK, d) if side == 0
                         else cells.view(kv, d, BLOCK).transpose(1, 2)).clone()
                grown = (now > was)[:, None, None]
                older = cells[:, :before] * (was / now_safe)[:, None, None]
                cells[:, :before] = torch.where(grown, _round64(older, codes.dtype), cells[:, :before])
                cells[:, before: before + hi - lo] = _round64(rows / now_safe[:, None, None], codes.dtype)
                cells[:, before + hi - lo:] = 0.0
                cells = (cells.view(kv, BLOCK, d // 16, 16).transpose(1, 2) if side == 0 else cells.transpose(1, 2))
                held[at, side, :, part] = cells.reshape(kv, BLOCK * d)
                scales[at, side, :, part] = now
    return {"q": q_out, "codes": held if codes.dtype != torch.int8 else None, "scales": scales}


def _round64(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The nearest number that an 8-bit code stands for, ties to even."""
    if dtype == torch.int8:
        return y.round()
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)  # three bits after the leading one, 2^-9 between subnormals
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def _exact_attend(case: dict, seed: int) -> torch.Tensor:
    """Sequence by sequence and head by head, the keys a sequence has and no others."""
    s = _state(case, seed)
    b, t, h, d = s["q"].shape
    kv, rep = case["kv_heads"], h // case["kv_heads"]
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=DEV)
    counts = [t] * b if s["new"] is None else s["new"].tolist()
    raw = s["codes"].view(torch.uint8)
    for n, start in enumerate(s["starts"].tolist()):
        length = start + counts[n]
        pages = s["table"][n, : -(-length // case["page"])].long()
        for j in range(kv):
            c = raw[pages, :, j].view(s["codes"].dtype).double() * s["scales"][pages, :, j].double()[..., None]
            keys = c[:, 0].unflatten(-1, (d // 16, BLOCK, 16)).permute(0, 1, 3, 2, 4).reshape(-1, d)[:length]
            values = c[:, 1].unflatten(-1, (d, BLOCK)).permute(0, 1, 3, 2).reshape(-1, d)[:length]
            rows = s["q"][n, : counts[n], j * rep: (j + 1) * rep].double()
            scores = rows.flatten(0, 1) @ keys.t().contiguous() / math.sqrt(d)
            seen = torch.arange(length, device=DEV) <= start + torch.arange(counts[n], device=DEV)[:, None]
            scores = scores.masked_fill(~seen.repeat_interleave(rep, 0), float("-inf"))
            mixed = torch.softmax(scores, -1) @ values.contiguous()
            out[n, : counts[n], j * rep: (j + 1) * rep] = mixed.unflatten(0, (counts[n], rep))
    return out


@torch.no_grad()
def exact(case: dict, seed: int):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "linear":
        s = _linear_inputs(case, seed)
        x = s["x"].double()
        scale = x.abs().amax(-1, keepdim=True) / 127.0
        codes = (x / scale).round()
        return (codes @ s["w"].double().t()) * scale * s["scale"].double()
    s = _copy_state(case, seed)  # a copy has nothing to round
    for src, dst in zip(s["src"], s["dst"]):
        s["codes"].view(torch.uint8)[:, dst] = s["codes"].view(torch.uint8)[:, src]
        s["scales"][:, dst] = s["scales"][:, src]
    return {"codes": s["codes"], "scales": s["scales"].double()}
