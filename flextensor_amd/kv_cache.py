"""A KV cache in pages of 8-bit codes, and the operations on it.

A decoder's cache is what grows with its users; in 8 bits it leaves twice the HBM of a bf16 cache to weights that
would otherwise stream. One layer is two tensors:

* ``codes`` [pages, 2, kv heads, blocks of a page, 32 * d], ``float8_e4m3fn`` or ``int8`` (-127 .. 127): the keys'
  side, then the values'. A block is 32 tokens of one head; its keys are stored as [d / 16, 32, 16], its values as
  [d, 32], the order in which the matrix cores take them.
* ``scales`` [pages, 2, kv heads, blocks of a page], fp32: a code ``c`` of a block stands for ``c * scale``.

:func:`append` rotates new queries and keys (normalised head by head first, where a model does so) and writes keys and
values, :func:`attention` attends over the cache, :func:`tree_attention` lets drafted tokens that form a tree attend over
it and their ancestors, :func:`keep` moves the accepted ones up, :func:`copy_pages` copies pages; each takes the
sequences' page ``table`` (int32; a number outside the pool is a hole whose tokens are not seen), the tokens that each has
cached (``starts``) and the new ones it adds (``new``) as device tensors, so a captured graph follows them.
:class:`PagedKVCache` owns the pool of all layers and its bookkeeping: sequences, shared pages, forks, drafted trees,
truncation and compaction.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _native as nat
from . import hip

BLOCK = nat.KV8_BLOCK
FORMATS = {torch.float8_e4m3fn: nat.KV8_E4M3, torch.int8: nat.KV8_INT8}
MAX_PAGE_TOKENS = 4096


_PLAIN = hip._PLAIN_TYPES
_Strides6 = ctypes.c_int64 * 6
_Strides9 = ctypes.c_int64 * 9


def _device(t: torch.Tensor) -> int:
    return torch._C._cuda_getDevice() if t.is_cuda else -2  # -1 is the host's


def _check_ints(what: str, name: str, t: torch.Tensor, dims: int, batch: int, device: int) -> None:
    if type(t) is not torch.Tensor or t.dtype != torch.int32:
        raise TypeError(f"{what} takes {name} as an int32 tensor")
    if t.dim() != dims or t.shape[0] != batch or t.get_device() != device:
        raise ValueError(f"{what} needs {name} of {batch} sequences on cuda:{device}, got {tuple(t.shape)} on {t.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1 or dims == 2 and batch > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what} needs {name} in rows that do not overlap, not of strides {t.stride()}")


def _check_pool(what: str, codes: torch.Tensor, scales: torch.Tensor, dims: int) -> None:
    for name, t in (("codes", codes), ("scales", scales)):
        if type(t) not in _PLAIN:
            raise TypeError(f"{what} takes plain tensors, {name} is a {type(t).__name__}")
    if codes.dtype not in FORMATS or scales.dtype != torch.float32:
        raise TypeError(f"{what} takes float8_e4m3fn or int8 codes and fp32 scales, got {codes.dtype} and {scales.dtype}")
    if codes.dim() != dims or codes.shape[:-1] != scales.shape or codes.shape[dims - 4] != 2:
        raise ValueError(f"{what}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are no pool of pages")
    if not hip._packed(codes, scales):
        raise ValueError(f"{what} needs contiguous, 16-byte aligned codes and scales")
    device = torch._C._cuda_getDevice() if codes.is_cuda else -1
    if device < 0 or codes.get_device() != device or scales.get_device() != device:
        raise ValueError(f"{what} runs on the current GPU, the cache is on {codes.device} and {scales.device}")
    page = codes.shape[-2] * BLOCK
    if codes.shape[-1] not in (64 * BLOCK, 128 * BLOCK) or page & (page - 1) or not BLOCK <= page <= MAX_PAGE_TOKENS:
        raise ValueError(f"{what}: pages hold 32 times a power of two tokens, up to {MAX_PAGE_TOKENS}, of 64 or 128 "
                         f"values each, not {tuple(codes.shape)}")


def _check_heads(what: str, **tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.dim() != 4:
            raise ValueError(f"{what} takes [batch, token, head, d] tensors, {name} is {tuple(t.shape)}")
    hip._check_operands(what, **tensors)
    for name, t in tensors.items():
        if hip._head_strides(t) is None:
            raise ValueError(f"{what} reads {name} 16 bytes at a time: it must be contiguous along d and 16-byte "
                             f"aligned, with strides that are multiples of 8, not {t.stride()}")


def _heads(what: str, device: int, *tensors: torch.Tensor) -> list[int]:
    """The strides of [batch, token, head, d] operands that the kernels can read (a call's q, k and v), else an error."""
    strides: list[int] = []
    grad = torch.is_grad_enabled()
    plain = torch.autograd.forward_ad._current_level < 0
    for t in tensors:
        if (type(t) not in _PLAIN or t.dtype is not torch.bfloat16 or t.dim() != 4 or t.get_device() != device
                or not plain or (grad and t.requires_grad)):
            _check_heads(what, **dict(zip("qkv", tensors)))
        got = hip._head_strides(t)
        if got is None:
            _check_heads(what, **dict(zip("qkv", tensors)))
        strides += got
    return strides


def _cache(what: str, q: torch.Tensor, device: int, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor,
           starts: torch.Tensor, new: torch.Tensor | None) -> nat.Kv8Cache:
    b, _, h, d = q.shape
    shape, dtype, i32 = codes.shape, codes.dtype, torch.int32
    ptr, scales_ptr = codes.data_ptr(), scales.data_ptr()
    if (type(codes) not in _PLAIN or type(scales) not in _PLAIN or dtype not in FORMATS or len(shape) != 5
            or scales.dtype is not torch.float32 or shape[:4] != scales.shape or shape[1] != 2
            or codes.get_device() != device or scales.get_device() != device or (ptr | scales_ptr) % 16
            or not codes.is_contiguous() or not scales.is_contiguous() or shape[4] not in (2048, 4096)
            or shape[3] & (shape[3] - 1) or not 1 <= shape[3] <= MAX_PAGE_TOKENS // BLOCK):
        _check_pool(what, codes, scales, 5)
    hip._check_underived(what, codes=codes, scales=scales)
    pages, _, kv, blocks, block_bytes = shape
    if block_bytes != BLOCK * d or h % kv:
        raise ValueError(f"{what}: queries {tuple(q.shape)} do not fit a cache of {kv} heads of {block_bytes // BLOCK}")
    if table.dtype is not i32 or starts.dtype is not i32 or table.dim() != 2 or starts.shape != (b,) or (
            table.get_device() != device or starts.get_device() != device or not starts.is_contiguous()
            or type(table) is not torch.Tensor or type(starts) is not torch.Tensor
            or table.shape[0] != b or not table.is_contiguous()):
        _check_ints(what, "table", table, 2, b, device)
        _check_ints(what, "starts", starts, 1, b, device)
    new_ptr = None
    if new is not None:
        if type(new) is not torch.Tensor or new.dtype is not i32 or new.shape != (b,) or new.get_device() != device or (
                not new.is_contiguous()):
            _check_ints(what, "new", new, 1, b, device)
        new_ptr = new.data_ptr()
    width = table.shape[1]
    return nat.Kv8Cache(ptr, scales_ptr, pages, table.data_ptr() or None, max(table.stride(0), width),
                        starts.data_ptr(), new_ptr, width, kv, blocks * BLOCK, d, FORMATS[dtype])


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
           new: torch.Tensor | None = None, *, positions: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
           k_norm: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Writes new tokens into the cache and returns the rotated queries, in one launch (``ftx_kv8_append``).

    ``q``, ``k``, ``v``: bf16 [batch, t, heads or kv heads, d]; ``cos``, ``sin``: fp32 [positions, d], both halves.
    Sequence b's token i (of ``new[b]``, None: t) gets position ``starts[b] + i``. A block's scale is the largest
    magnitude of its tokens over 448 (e4m3) or 127 (int8); it only grows while the block fills, and the block's
    older codes are rounded again when it does. Sequences with a negative start, tokens past the table or the rotary
    positions, and holes are left out; the queries of tokens left out are 0. :func:`attention` has no positions: it
    would see the places of tokens past the rotary tables. Two sequences of a call must not write into one page.

    ``q_norm``, ``k_norm``: bf16 [d]; queries and keys are first normalised head by head, ``x / sqrt(mean(x^2) + eps)``
    times these, in the same launch (``ftx_kv8_append_norm``). ``positions``: int32 [batch, t], the rows of the rotary
    tables that tokens are turned by in place of their places' (nodes of a tree: the prefix's length and their depth); a
    token of a position outside the tables becomes 0, in the cache too, and must not be attended to.
    """
    device = _device(q)
    plain = positions is None and q_norm is None and k_norm is None
    if device >= 0 and torch.autograd.forward_ad._current_level < 0:
        stream = hip._stream(device)
        if plain:
            got = nat.torch_calls().append(q, k, v, cos, sin, codes, scales, table, starts, new, device, stream)
        else:
            got = nat.torch_calls().append_norm(q, k, v, cos, sin, codes, scales, table, starts, new, positions, q_norm,
                                                k_norm, eps, device, stream)
        if got is not None:
            return nat.result(got)
    strides = _heads("append", device, q, k, v)
    cache = _cache("append", q, device, codes, scales, table, starts, new)
    b, t, h, d = shape = q.shape
    if k.shape != (b, t, cache.kv_heads, d) or v.shape != k.shape:
        raise ValueError(f"append operands differ: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} for "
                         f"{cache.kv_heads} cached heads")
    cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    for name, x in (("cos", cos), ("sin", sin)):
        if type(x) not in _PLAIN or x.dtype is not torch.float32:
            raise TypeError(f"append takes {name} as an fp32 tensor")
        if x.dim() != 2 or x.shape != cos.shape or x.shape[1] != d or x.get_device() != device or not x.is_contiguous() or (
                (cos_ptr | sin_ptr) % 16):
            raise ValueError(f"append needs cos and sin [positions, {d}], contiguous, 16-byte aligned and on {q.device}")
    hip._check_underived("append", cos=cos, sin=sin)
    if (q_norm is None) != (k_norm is None):
        raise ValueError("append takes norm weights for both q and k, or none")
    if q_norm is not None:
        hip._check_operands("append", q_norm=q_norm, k_norm=k_norm)
        if q_norm.shape != (d,) or k_norm.shape != (d,) or not hip._packed(q_norm, k_norm):
            raise ValueError(f"append needs norm weights [{d}], contiguous and 16-byte aligned, got {tuple(q_norm.shape)} "
                             f"and {tuple(k_norm.shape)}")
        if not 0.0 <= eps < float("inf"):
            raise ValueError(f"append needs a finite eps that is not negative, not {eps}")
    if positions is not None:
        _check_ints("append", "positions", positions, 2, b, device)
        if positions.shape[1] != t:
            raise ValueError(f"append needs a position for each of {t} tokens, got {tuple(positions.shape)}")
    torch._C._increment_version((codes, scales))  # as an in-place operation, for what autograd saved
    out = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    if not plain:
        nat.call("ftx_kv8_append_norm", ctypes.byref(cache), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                 *[w.data_ptr() if w is not None else None for w in (q_norm, k_norm)], eps, cos_ptr, sin_ptr, cos.shape[0],
                 (positions.data_ptr() or None) if positions is not None else None,
                 max(positions.stride(0), t) if positions is not None else 0, out.data_ptr(), b, t, h,
                 _Strides9(*strides), hip._stream(device))
        return out
    nat.call("ftx_kv8_append", ctypes.byref(cache), q.data_ptr(), k.data_ptr(), v.data_ptr(), cos_ptr, sin_ptr,
             cos.shape[0], out.data_ptr(), b, t, h, _Strides9(*strides), hip._stream(device))
    return out


def attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
              new: torch.Tensor | None = None, max_tokens: int | None = None,
              scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of new tokens over the cache, each over the tokens up to its own
    (``ftx_kv8_attention``).

    ``q``: bf16 [batch, t, heads, d], rotated; its tokens are in the cache. Token i of sequence b (of ``new[b]``,
    None: t) sees positions up to ``starts[b] + i``; the result of a token left out, or that sees nothing, is 0.
    ``max_tokens``: the longest sequence, new tokens included (None: all that the table holds). It shapes the launch
    and changes no result beyond the order of the sums and, for more than 64 rows (tokens times the heads that share a
    cached one), the rounding of the probabilities: prompts in tiles of 256 rows round each to bf16 for the matrix cores
    (0.0024 of the result in relative norm, 0.0017 being the output's own rounding), fewer rows do not. ``scale``:
    1 / sqrt(d) if None. A NaN that a sequence holds may reach earlier tokens of the same call. The sums are fp32: values
    of up to about 1e30 stay finite.
    """
    device = _device(q)
    if device >= 0 and torch.autograd.forward_ad._current_level < 0:
        got = nat.torch_calls().attention(q, codes, scales, table, starts, new, max_tokens, scale, device,
                                          hip._stream(device))
        if got is not None:
            return nat.result(got)
    strides = _heads("attention", device, q)
    cache = _cache("attention", q, device, codes, scales, table, starts, new)
    b, t, h, d = q.shape
    longest = cache.width * cache.page_tokens
    if max_tokens is not None:
        if max_tokens < 0:
            raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
        longest = min(longest, max_tokens)
    out = torch.empty_like(q)
    strides += hip._head_strides(out)
    got = ctypes.c_size_t(0)
    nat.call("ftx_kv8_attention_workspace", b, t, h, cache.kv_heads, d, longest, ctypes.byref(got))
    ws_bytes = int(got.value)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    nat.call("ftx_kv8_attention", ctypes.byref(cache), q.data_ptr(), out.data_ptr(), b, t, h,
             _Strides6(*strides), d ** -0.5 if scale is None else scale, longest,
             ws.data_ptr() if ws is not None else None, ws_bytes, hip._stream(device))
    return out


def tree_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                   tree: torch.Tensor, new: torch.Tensor | None = None, *, nodes: int | None = None,
                   max_tokens: int | None = None, scale: float | None = None) -> torch.Tensor:
    """:func:`attention` of drafted tokens that form a tree (``ftx_kv8_tree_attention``).

    ``starts[b]``: the first tokens of a sequence, which every row sees. The ``nodes`` tokens (None: t; at most 64) cached
    after them are the tree's nodes, and ``tree`` (int64 [batch, t]) says which of them a row sees: bit j of
    ``tree[b, i]`` the token ``starts[b] + j`` (one tree may be expanded over the batch). A row's own node is one of its
    bits, its ancestors the others; rows may be a part of the nodes (a level of the tree). Rows from ``new[b]`` on, and
    rows that see no token, are 0. Nodes behind the last one that a row of the sequence sees, and blocks of 32 tokens of
    which none sees one, may hold anything: they need not have been written. A NaN that another node's value holds may
    reach rows that do not see it. ``max_tokens`` counts the nodes. Many rows are shared out by the lengths of the whole
    batch, which may change the order of a sum.
    """
    device = _device(q)
    if device >= 0 and torch.autograd.forward_ad._current_level < 0:
        got = nat.torch_calls().tree_attention(q, codes, scales, table, starts, tree, new, nodes, max_tokens, scale, device,
                                               hip._stream(device))
        if got is not None:
            return nat.result(got)
    strides = _heads("tree_attention", device, q)
    cache = _cache("tree_attention", q, device, codes, scales, table, starts, new)
    b, t, h, d = q.shape
    if type(tree) is not torch.Tensor or tree.dtype != torch.int64:
        raise TypeError("tree_attention takes tree as an int64 tensor")
    if tree.shape != (b, t) or tree.get_device() != device or (t > 1 and tree.stride(1) != 1) or (
            b > 1 and tree.stride(0) != 0 and tree.stride(0) < t):
        raise ValueError(f"tree_attention needs a set of nodes for each of [{b}, {t}] rows on cuda:{device}, in rows that do "
                         f"not overlap, got {tuple(tree.shape)} of strides {tree.stride()} on {tree.device}")
    nodes = t if nodes is None else nodes
    if not 0 <= nodes <= nat.KV8_TREE_NODES:
        raise ValueError(f"a tree has 0 to {nat.KV8_TREE_NODES} nodes, not {nodes}")
    longest = cache.width * cache.page_tokens
    if max_tokens is not None:
        if max_tokens < 0:
            raise ValueError(f"max_tokens must not be negative, got {max_tokens}")
        longest = min(longest, max_tokens)
    out = torch.empty_like(q)
    strides += hip._head_strides(out)
    got = ctypes.c_size_t(0)
    nat.call("ftx_kv8_tree_attention_workspace", b, t, h, cache.kv_heads, d, longest, ctypes.byref(got))
    ws_bytes = int(got.value)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    nat.call("ftx_kv8_tree_attention", ctypes.byref(cache), q.data_ptr(), out.data_ptr(), tree.data_ptr(),
             tree.stride(0) if b > 1 else t, nodes, b, t, h, _Strides6(*strides), d ** -0.5 if scale is None else scale,
             longest, ws.data_ptr() if ws is not None else None, ws_bytes, hip._stream(device))
    return out


def keep(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, path: torch.Tensor,
         counts: torch.Tensor | None = None) -> None:
    """Moves the accepted nodes of drafted trees behind their sequences' first tokens, in every layer of a pool
    [layers, pages, ...], in one launch (``ftx_kv8_keep``).

    Token ``starts[b] + path[b, i]`` moves to ``starts[b] + i``, for i below ``counts[b]`` (None: all of path's n, at most
    64). ``path``: int32 [batch, n], ascending; it ends before an entry that does not ascend or is 64 or more. Keys and
    values stay what they are, but for tokens that move into a block of another scale: a block's scale becomes the largest
    that its tokens had, and codes of another one are rounded again. What lies behind the last kept token of its block
    becomes 0. Two sequences must not write into one page.
    """
    device = _device(codes)
    if device >= 0 and torch.autograd.forward_ad._current_level < 0:
        got = nat.torch_calls().keep(codes, scales, table, starts, path, counts, device, hip._stream(device))
        if got is not None:
            nat.result(got)
            return
    _check_pool("keep", codes, scales, 6)
    hip._check_underived("keep", codes=codes, scales=scales)
    if path.dim() != 2:
        raise ValueError(f"keep takes a path [batch, n], got {tuple(path.shape)}")
    b, n = path.shape
    _check_ints("keep", "path", path, 2, b, device)
    _check_ints("keep", "table", table, 2, b, device)
    _check_ints("keep", "starts", starts, 1, b, device)
    if counts is not None:
        _check_ints("keep", "counts", counts, 1, b, device)
    if n > nat.KV8_TREE_NODES:
        raise ValueError(f"keep moves up to {nat.KV8_TREE_NODES} nodes of a sequence, not {n}")
    layers, pages, _, kv, blocks, block_bytes = codes.shape
    torch._C._increment_version((codes, scales))
    if not layers:
        return
    width = table.shape[1]
    cache = nat.Kv8Cache(codes.data_ptr(), scales.data_ptr(), pages, table.data_ptr() or None, max(table.stride(0), width),
                         starts.data_ptr(), counts.data_ptr() if counts is not None else None, width, kv, blocks * BLOCK,
                         block_bytes // BLOCK, FORMATS[codes.dtype])
    nat.call("ftx_kv8_keep", ctypes.byref(cache), layers, path.data_ptr(), max(path.stride(0), n), b, n, hip._stream(device))


def copy_pages(codes: torch.Tensor, scales: torch.Tensor, src: list[int], dst: list[int]) -> None:
    """Copies pages ``src[i]`` to ``dst[i]`` in every layer of a pool, [layers, pages, ...] codes and scales
    (``ftx_kv8_copy_pages``). No page is written twice or both read and written. The numbers travel with the launch:
    nothing is uploaded."""
    device = _device(codes)
    if device >= 0 and torch.autograd.forward_ad._current_level < 0:
        got = nat.torch_calls().copy_pages(codes, scales, src, dst, device, hip._stream(device))
        if got is not None:
            nat.result(got)
            return
    _check_pool("copy_pages", codes, scales, 6)
    hip._check_underived("copy_pages", codes=codes, scales=scales)
    if len(src) != len(dst):
        raise ValueError(f"copy_pages takes as many sources as targets, got {len(src)} and {len(dst)}")
    layers, pages, _, kv, blocks, block_bytes = codes.shape
    if src and not 0 <= min(min(src), min(dst)) <= max(max(src), max(dst)) < pages:  # before they become 32-bit
        raise ValueError(f"copy_pages: a page number outside the pool of {pages}")
    torch._C._increment_version((codes, scales))
    n = len(src)
    nat.call("ftx_kv8_copy_pages", codes.data_ptr(), scales.data_ptr(), layers, pages, kv, blocks * BLOCK,
             block_bytes // BLOCK, (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, hip._stream())


def read(codes: torch.Tensor, scales: torch.Tensor, table: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that pages stand for, fp32 [..., tokens, kv heads, d] for a table [..., pages] of one
    layer (torch operations: for inspection and export, not for a step). Holes are zeros."""
    d, blocks, kv = codes.shape[-1] // BLOCK, codes.shape[-2], codes.shape[-3]
    hole = (table < 0) | (table >= codes.shape[0])
    table = table.long().masked_fill(hole, 0)
    c = codes.view(torch.uint8)[table].view(codes.dtype).float() * scales[table].unsqueeze(-1)
    c = c.masked_fill_(hole.view(*hole.shape, *[1] * 4), 0.0)
    lead = table.shape[:-1]
    c = c.movedim(-4, 0)  # [2, ..., pages, kv, blocks, 32 d]
    keys = c[0].unflatten(-1, (d // 16, BLOCK, 16)).transpose(-3, -2).flatten(-2)
    values = c[1].unflatten(-1, (d, BLOCK)).transpose(-2, -1)
    return tuple(x.movedim(-4, -2).reshape(*lead, table.shape[-1] * blocks * BLOCK, kv, d) for x in (keys, values))


class KVCacheFull(RuntimeError):
    """The pool has too few free pages for a request; nothing has been changed."""


@dataclass(frozen=True)
class KVStep:
    """The sequences of one forward pass: what every layer's calls share. :meth:`layer` is one layer's cache."""

    cache: "PagedKVCache"
    sequences: tuple[int, ...]
    counts: tuple[int, ...]
    table: torch.Tensor
    starts: torch.Tensor
    new: torch.Tensor
    tokens: int
    max_tokens: int
    held: tuple = ()  # of each sequence: its length, and the pages that its new tokens go to
    moves: int = 0  # compactions of the cache before it
    most: int = 0  # the largest count

    def layer(self, index: int) -> "KVLayer":
        return KVLayer(self, index)

    def check(self, batch: int, tokens: int, positions: int) -> None:
        """Refuses a pass of [batch, tokens] rows that does not hold the step's tokens, or whose rotary tables of so
        many ``positions`` end before them."""
        if batch != len(self.sequences) or tokens < self.most:
            raise ValueError(f"the step counts {self.counts} tokens of {len(self.sequences)} sequences, the pass has "
                             f"{tokens} of {batch}")
        if self.max_tokens > positions and any(c and was[0] + c > positions for c, was in zip(self.counts, self.held)):
            raise ValueError(f"the step's sequences grow to {self.max_tokens} tokens, the model has {positions} positions")


@dataclass(frozen=True)
class KVLayer:
    """One layer of the cache in a step: :meth:`append`, then :meth:`attend`."""

    step: KVStep
    index: int

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               **norms) -> torch.Tensor:
        """``norms``: q_norm, k_norm and eps of :func:`append`."""
        s = self.step
        s.check(q.shape[0], q.shape[1], cos.shape[0])
        return append(q, k, v, cos, sin, s.cache.codes[self.index], s.cache.scales[self.index], s.table, s.starts, s.new,
                      **norms)

    def attend(self, q: torch.Tensor) -> torch.Tensor:
        s = self.step
        return attention(q, s.cache.codes[self.index], s.cache.scales[self.index], s.table, s.starts, s.new,
                         max_tokens=s.max_tokens)


@dataclass(frozen=True)
class KVTree:
    """Drafted tokens behind the cached ones of some sequences, a tree of one shape each: what the passes over them share.
    :meth:`nodes` is the step of some of the nodes."""

    cache: "PagedKVCache"
    step: KVStep  # of all the nodes, as if they were a chain
    parents: tuple[int, ...]
    depths: tuple[int, ...]
    sets: torch.Tensor  # int64 [1, nodes]: the nodes that each one sees
    starts: torch.Tensor  # int32 [nodes, batch]: how many first tokens and nodes come before each
    positions: torch.Tensor  # int32 [batch, nodes]

    def nodes(self, first: int = 0, last: int | None = None) -> "KVNodes":
        """The step of nodes ``first`` .. ``last - 1`` (None: all that follow); the ones before are in the cache."""
        last = len(self.parents) if last is None else last
        if not 0 <= first < last <= len(self.parents):
            raise ValueError(f"nodes {first} to {last} of a tree of {len(self.parents)}")
        return KVNodes(self, first, last)

    def levels(self) -> list[tuple[int, int]]:
        """The nodes of each depth as ranges, where the tree lists them so."""
        if list(self.depths) != sorted(self.depths):
            raise ValueError("the tree does not list its nodes level by level")
        return [(self.depths.index(d), self.depths.index(d) + self.depths.count(d)) for d in sorted(set(self.depths))]


@dataclass(frozen=True)
class KVNodes:
    """Some nodes of drafted trees as the step of a forward pass."""

    tree: KVTree
    first: int
    last: int

    @property
    def counts(self) -> tuple[int, ...]:
        return (self.last - self.first,) * len(self.tree.step.sequences)

    def layer(self, index: int) -> "KVTreeLayer":
        return KVTreeLayer(self, index)

    def check(self, batch: int, tokens: int, positions: int) -> None:
        """Refuses a pass of [batch, tokens] rows that are not the nodes, or whose rotary tables end before them."""
        step = self.tree.step
        if (batch, tokens) != (len(step.sequences), self.last - self.first):
            raise ValueError(f"the step has nodes {self.first} to {self.last} of {len(step.sequences)} trees, the pass "
                             f"{tokens} of {batch}")
        deepest = max((was[0] for was in step.held), default=0) + max(self.tree.depths[self.first: self.last])
        if deepest >= positions:
            raise ValueError(f"the trees reach position {deepest}, the model has {positions}")


@dataclass(frozen=True)
class KVTreeLayer(KVLayer):
    """One layer of the cache in a step of a tree's nodes."""

    step: KVNodes

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               **norms) -> torch.Tensor:
        s, t = self.step, self.step.tree
        s.check(q.shape[0], q.shape[1], cos.shape[0])
        return append(q, k, v, cos, sin, t.cache.codes[self.index], t.cache.scales[self.index], t.step.table,
                      t.starts[s.first], positions=t.positions[:, s.first: s.last], **norms)

    def attend(self, q: torch.Tensor) -> torch.Tensor:
        s, t = self.step, self.step.tree
        return tree_attention(q, t.cache.codes[self.index], t.cache.scales[self.index], t.step.table, t.starts[0],
                              t.sets[:, s.first: s.last].expand(q.shape[0], -1), nodes=s.last,
                              max_tokens=t.step.max_tokens - len(t.parents) + s.last)


class PagedKVCache:
    """The pages of all layers, and which sequence holds which.

    A sequence is a number from :meth:`open`. :meth:`begin` reserves pages for its next tokens and returns the
    :class:`KVStep` that the layers' calls take; :meth:`commit` counts those tokens as cached once the pass has been
    queued. :meth:`fork` gives a sequence's pages to another one too: full pages stay shared, and the page that one
    of them writes into next is copied first. :meth:`draft` reserves pages for a tree of drafted tokens behind each
    sequence, and :meth:`accept` keeps one path of each. :meth:`truncate` drops a sequence's last tokens, :meth:`close`
    all of it. :meth:`compact` moves the pages in use to the pool's start and :meth:`resize` then gives the rest back.

    The bookkeeping is the host's; every device operation runs on torch's current stream, which must be the same
    one, or ordered, from call to call.
    """

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page_tokens: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device: torch.device | str = "cuda") -> None:
        if layers < 1 or kv_heads < 1 or pages < 1:
            raise ValueError(f"a cache needs layers, heads and pages, got {layers}, {kv_heads} and {pages}")
        if head_dim not in (64, 128):
            raise ValueError(f"the 8-bit cache holds head dimensions 64 and 128, not {head_dim}")
        if page_tokens & (page_tokens - 1) or not BLOCK <= page_tokens <= MAX_PAGE_TOKENS:
            raise ValueError(f"a page holds 32 times a power of two tokens, up to {MAX_PAGE_TOKENS}, not {page_tokens}")
        if dtype not in FORMATS:
            raise TypeError(f"cache codes are float8_e4m3fn or int8, not {dtype}")
        self.layers, self.kv_heads, self.head_dim = layers, kv_heads, head_dim
        self.page_tokens, self.dtype, self.device = page_tokens, dtype, torch.device(device)
        self.codes, self.scales = self._tensors(pages)
        self._free = list(range(pages - 1, -1, -1))  # taken from the end: the lowest number first
        self._refs = [0] * pages
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0
        self._moves = 0

    def _tensors(self, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
        shape = (self.layers, pages, 2, self.kv_heads, self.page_tokens // BLOCK)
        codes = torch.empty((*shape, BLOCK * self.head_dim), dtype=self.dtype, device=self.device)
        codes.view(torch.uint8).zero_()
        return codes, torch.zeros(shape, dtype=torch.float32, device=self.device)

    @property
    def pages(self) -> int:
        return self.codes.shape[1]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def page_bytes(self) -> int:
        """Bytes of one page in all layers."""
        return self.layers * 2 * self.kv_heads * (self.page_tokens * self.head_dim + 4 * self.page_tokens // BLOCK)

    def length(self, sequence: int) -> int:
        return self._lengths[sequence]

    def table(self, sequence: int) -> list[int]:
        """The pages of a sequence, in order."""
        return list(self._pages[sequence])

    def open(self) -> int:
        """A new, empty sequence."""
        sequence, self._next = self._next, self._next + 1
        self._pages[sequence], self._lengths[sequence] = [], 0
        return sequence

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens, on the same pages. Pages that a step not committed has reserved stay
        the sequence's own."""
        length = self._lengths[sequence]
        pages = self._pages[sequence][: -(-length // self.page_tokens)]
        other = self.open()
        for p in pages:
            self._refs[p] += 1
        self._pages[other], self._lengths[other] = pages, length
        return other

    def truncate(self, sequence: int, length: int) -> None:
        """Keeps the first ``length`` tokens. A block that is cut keeps its scale."""
        if not 0 <= length <= self._lengths[sequence]:
            raise ValueError(f"sequence {sequence} holds {self._lengths[sequence]} tokens, {length} cannot be kept")
        pages = self._pages[sequence]
        keep = -(-length // self.page_tokens)
        for p in pages[keep:]:
            self._drop(p)
        del pages[keep:]
        self._lengths[sequence] = length

    def close(self, sequence: int) -> None:
        """Drops a sequence; pages that no other one holds are free again."""
        self.truncate(sequence, 0)
        del self._pages[sequence], self._lengths[sequence]

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if not self._refs[page]:
            self._free.append(page)

    def _take(self) -> int:
        page = self._free.pop()
        self._refs[page] = 1
        return page

    def begin(self, sequences: list[int], counts: list[int] | int, tokens: int | None = None) -> KVStep:
        """Reserves pages for ``counts[i]`` more tokens of ``sequences[i]``. ``tokens``: the row length of the pass
        (None: the largest count). A page that would be written and is shared is copied first."""
        counts = [counts] * len(sequences) if isinstance(counts, int) else list(counts)
        if len(counts) != len(sequences) or len(set(sequences)) != len(sequences):
            raise ValueError("a step takes different sequences and a count for each")
        tokens = max(counts, default=0) if tokens is None else tokens
        if any(not 0 <= c <= tokens for c in counts):
            raise ValueError(f"counts {counts} outside [0, {tokens}]")
        size = self.page_tokens
        need, shared = 0, []
        sharers: dict[int, int] = {}  # what is left of a shared page's references as this step's sequences leave it
        for s, c in zip(sequences, counts):
            length, held = self._lengths[s], self._pages[s]
            end = -(-(length + c) // size)
            need += max(0, end - len(held))
            for at in range(length // size, min(end, len(held)) if c else 0):  # held pages that the step writes
                left = sharers.setdefault(held[at], self._refs[held[at]])
                if left > 1:
                    sharers[held[at]] = left - 1
                    shared.append((s, at))
        if need + len(shared) > len(self._free):
            raise KVCacheFull(f"{need + len(shared)} pages needed, {len(self._free)} of {self.pages} free")
        src = [self._pages[s][at] for s, at in shared]
        if src:  # a copy that fails leaves the books as they were
            copy_pages(self.codes, self.scales, src, self._free[: -len(src) - 1: -1])
        for (s, at), old in zip(shared, src):
            self._pages[s][at] = self._take()
            self._refs[old] -= 1
        for s, c in zip(sequences, counts):
            held = self._pages[s]
            while len(held) * size < self._lengths[s] + c:
                held.append(self._take())
        b = len(sequences)
        width = max((len(self._pages[s]) for s in sequences), default=0)
        rows = [p for s in sequences for p in self._pages[s] + [-1] * (width - len(self._pages[s]))]
        host = torch.tensor([self._lengths[s] for s in sequences] + counts + rows, dtype=torch.int32)
        dev = host.to(self.device)  # one upload
        longest = max((self._lengths[s] + c for s, c in zip(sequences, counts)), default=0)
        return KVStep(self, tuple(sequences), tuple(counts), dev[2 * b:].view(b, width), dev[:b], dev[b: 2 * b],
                      tokens, longest, tuple(self._state(s, c) for s, c in zip(sequences, counts)), self._moves,
                      max(counts, default=0))

    def _state(self, sequence: int, count: int) -> tuple[int, list[int]]:
        """The length of a sequence, and the pages that its next tokens go to."""
        length, size = self._lengths[sequence], self.page_tokens
        return length, self._pages[sequence][length // size: -(-(length + count) // size) if count else 0]

    def commit(self, step: KVStep) -> None:
        """Counts a step's tokens as cached. A step counts once, and only where its sequences are as they were when it
        began: not truncated or closed, and the pages that it wrote still theirs (or moved by :meth:`compact`)."""
        self._check_step(step)
        for s, c in zip(step.sequences, step.counts):
            self._lengths[s] += c

    def _check_step(self, step: KVStep) -> None:
        def changed(sequence: int, count: int, was: tuple[int, list[int]]) -> bool:
            if self._lengths.get(sequence) != was[0]:
                return True
            now = self._state(sequence, count)
            return now != was if step.moves == self._moves else len(now[1]) != len(was[1])  # moved: as many pages

        if step.cache is not self or any(map(changed, step.sequences, step.counts, step.held)):
            raise ValueError("the step was committed before, or its sequences have changed since it began")

    def draft(self, sequences: list[int], parents: list[int]) -> KVTree:
        """Reserves pages for a tree of drafted tokens behind each sequence. ``parents[i]``: the node before node i, a
        lower number, or -1 for one that follows the cached tokens; 64 nodes at most. A node sees the cached tokens, its
        ancestors and itself, and has the position that its depth gives it."""
        parents = list(parents)
        n, b = len(parents), len(sequences)
        if not 1 <= n <= nat.KV8_TREE_NODES or any(not -1 <= p < i for i, p in enumerate(parents)):
            raise ValueError(f"a tree has 1 to {nat.KV8_TREE_NODES} nodes, each behind its parent, got {parents}")
        sets, depths = [], []
        for i, p in enumerate(parents):
            sets.append(1 << i | (sets[p] if p >= 0 else 0))
            depths.append(depths[p] + 1 if p >= 0 else 0)
        step = self.begin(sequences, n)
        lengths = [self._lengths[s] for s in sequences]
        host = torch.tensor([x + d for x in lengths for d in depths] + [x + i for i in range(n) for x in lengths],
                            dtype=torch.int32)
        masks = torch.tensor([[s - (1 << 64) if s >> 63 else s for s in sets]], dtype=torch.int64)
        at = host.to(self.device)
        return KVTree(self, step, tuple(parents), tuple(depths), masks.to(self.device), at[b * n:].view(n, b),
                      at[: b * n].view(b, n))

    def accept(self, tree: KVTree, paths: list[list[int]]) -> None:
        """Counts one path of each tree as cached, in the order of its nodes (each the child of the one before; empty:
        none), and moves its keys and values to follow the sequence's tokens. Conditions as for :meth:`commit`."""
        step = tree.step
        if len(paths) != len(step.sequences):
            raise ValueError(f"{len(paths)} paths for {len(step.sequences)} sequences")
        for path in paths:
            if any(not 0 <= n < len(tree.parents) or tree.parents[n] != before for n, before in zip(path, [-1, *path])):
                raise ValueError(f"{path} is no path of the tree {list(tree.parents)}")
        self._check_step(step)
        b, n, width = len(paths), max(map(len, paths), default=0), step.table.shape[1]
        if any(path != list(range(len(path))) for path in paths):  # others are where they belong
            pages = [p for s in step.sequences  # as they are now: compact may have moved them
                     for p in self._pages[s][:width] + [-1] * (width - len(self._pages[s]))]
            host = torch.tensor([len(p) for p in paths] + [x for p in paths for x in [*p, *[0] * (n - len(p))]] + pages,
                                dtype=torch.int32)
            dev = host.to(self.device)  # one upload
            keep(self.codes, self.scales, dev[b + b * n:].view(b, width), tree.starts[0], dev[b: b + b * n].view(b, n),
                 dev[:b])
        for s, path in zip(step.sequences, paths):
            self._lengths[s] += len(path)

    def compact(self) -> int:
        """Moves pages in use to the pool's start, the fewest that leave no free page before them, and returns how
        many moved. Steps begun before hold stale tables."""
        used = self.pages - len(self._free)
        src = [p for p in range(used, self.pages) if self._refs[p]]
        dst = [p for p in range(used) if not self._refs[p]]
        if src:
            copy_pages(self.codes, self.scales, src, dst)
            to = dict(zip(src, dst))
            for s, d in to.items():
                self._refs[d], self._refs[s] = self._refs[s], 0
            for pages in self._pages.values():
                pages[:] = [to.get(p, p) for p in pages]
            self._moves += 1
        self._free = list(range(self.pages - 1, used - 1, -1))
        return len(src)

    def resize(self, pages: int) -> None:
        """Changes the number of pages; those in use must be among the first ``pages`` (:meth:`compact`). The pool is
        other tensors then: what holds the old ones (a captured graph) does not follow."""
        if pages < 1 or any(self._refs[pages:]):
            raise ValueError(f"a pool of {pages} pages does not hold the pages in use")
        codes, scales = self._tensors(pages)
        n = min(pages, self.pages)
        codes.view(torch.uint8)[:, :n] = self.codes.view(torch.uint8)[:, :n]
        scales[:, :n] = self.scales[:, :n]
        self.codes, self.scales = codes, scales
        self._refs = self._refs[:n] + [0] * (pages - n)
        self._free = [p for p in range(pages - 1, -1, -1) if not self._refs[p]]
