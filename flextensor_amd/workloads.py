"""Synthetic, seeded workloads that exercise the streaming path.

* :func:`build_mlp_stack` - n x [Linear(h -> i, bias) -> SiLU -> Linear(i -> h, bias)]
  (8 layers at 4096 -> 11008 -> 4096 for the MLP-stack workload).
* :class:`LlamaModel` - Llama-style decoder: RMSNorm, rotary attention with a
  KV cache, SwiGLU MLP (32 layers, hidden 4096, 32 x 128 heads, 11008
  intermediate, vocab 32000 for the 7B shape).
* :func:`scatter_tensor_set` - the tensor set of the scatter microbenchmark:
  byte sizes log-uniform in [4 KiB, 64 MiB], bf16, 1-D or 2-D shapes.

Weights are drawn N(0, 0.02) in float32 from one ``torch.Generator`` seeded
with ``seed``, parameter by parameter in module registration order, then
cast to bfloat16. ``init_device="cuda"`` draws on the device generator (fast
for multi-GB models) and copies the result into CPU tensors; the two devices
give different (each deterministic) weights.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch
import torch.nn.functional as F
from torch import nn
from torch.nn.modules import module as torch_module

from . import hip, kv_cache


FP8_E4M3_MAX = 448.0
INT8_MAX = 127.0


def init_normal_(model: nn.Module, seed: int, std: float = 0.02, init_device: str = "cpu") -> nn.Module:
    """Overwrite every parameter with N(0, std) draws (float32, then cast).

    An ``Fp8Linear`` draws its weight the same way, then stores it as
    float8_e4m3fn with a per-output-channel scale ``absmax / 448`` (bf16); the
    quantised weight is ``round_e4m3(w / scale)``. An ``Int8Linear``'s is
    ``round(w / scale)`` with ``absmax / 127`` (fp32), an ``Int4Linear``'s the
    same with ``absmax / 7`` of each group of inputs (bf16).
    """
    gen = torch.Generator(device=init_device).manual_seed(seed)
    with torch.no_grad():
        for mod in model.modules():
            if isinstance(mod, Fp8Linear):
                w = torch.empty(mod.weight.shape, dtype=torch.float32, device=init_device)
                w.normal_(0.0, std, generator=gen)
                scale = (w.abs().amax(dim=1) / FP8_E4M3_MAX).clamp_min(1e-12).to(torch.bfloat16)
                mod.weight.copy_((w / scale.float()[:, None]).to(torch.float8_e4m3fn))
                mod.scale.copy_(scale)
                continue
            if isinstance(mod, Int8Linear):
                w = torch.empty(mod.weight.shape, dtype=torch.float32, device=init_device)
                w.normal_(0.0, std, generator=gen)
                scale = (w.abs().amax(dim=1) / INT8_MAX).clamp_min(1e-12)
                mod.weight.copy_((w / scale[:, None]).round().to(torch.int8))
                mod.scale.copy_(scale)
                continue
            if isinstance(mod, Int4Linear):
                w = torch.empty(mod.out_features, mod.in_features, dtype=torch.float32, device=init_device)
                mod.quantize_(w.normal_(0.0, std, generator=gen))
                continue
            for p in mod.parameters(recurse=False):
                w = torch.empty(p.shape, dtype=torch.float32, device=init_device)
                w.normal_(0.0, std, generator=gen)
                p.copy_(w.to(p.dtype))
    return model


class MLPBlock(nn.Module):
    def __init__(self, hidden: int, inter: int, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.fc1 = nn.Linear(hidden, inter, bias=True, dtype=dtype)
        self.fc2 = nn.Linear(inter, hidden, bias=True, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.fc2(F.silu(self.fc1(x)))


class MLPStack(nn.Module):
    def __init__(self, n_layers: int, hidden: int, inter: int, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.layers = nn.ModuleList(MLPBlock(hidden, inter, dtype) for _ in range(n_layers))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for layer in self.layers:
            x = layer(x)
        return x


def build_mlp_stack(n_layers: int = 8, hidden: int = 4096, inter: int = 11008, seed: int = 0,
                    init_device: str = "cpu") -> MLPStack:
    with torch.device("meta"):
        model = MLPStack(n_layers, hidden, inter)
    model = model.to_empty(device="cpu")
    return init_normal_(model, seed, 0.02, init_device)


def mlp_input(batch: int = 16, hidden: int = 4096, seed: int = 0) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(batch, hidden, generator=gen, dtype=torch.float32).to(torch.bfloat16)


# ---- Llama-style decoder -----------------------------------------------------


@dataclass(frozen=True)
class LlamaShape:
    n_layers: int = 32
    hidden: int = 4096
    n_heads: int = 32
    n_kv_heads: int = 32
    head_dim: int = 128
    inter: int = 11008
    vocab: int = 32000
    max_seq: int = 2048
    eps: float = 1e-5
    rope_theta: float = 10000.0
    fp8: bool = False  # projection weights in float8_e4m3fn with per-output-channel bf16 scales
    int8: bool = False  # projection weights and their inputs in 8-bit integers, fp32 scales per channel and per token
    int4: bool = False  # projection weights in 4 bits with bf16 scales for groups of a channel's inputs
    qk_norm: bool = False  # queries and keys normalised head by head before they are rotated

    def layer_bytes(self, itemsize: int = 2) -> int:
        h, d = self.hidden, self.head_dim
        mats = h * self.n_heads * d + 2 * h * self.n_kv_heads * d + self.n_heads * d * h + 3 * h * self.inter
        norms = 2 * h + (2 * d if self.qk_norm else 0)
        if self.int4:
            shapes = [(h, self.n_heads * d), *[(h, self.n_kv_heads * d)] * 2, (self.n_heads * d, h),
                      *[(h, self.inter)] * 2, (self.inter, h)]
            return sum(Int4Linear.nbytes(*shape) for shape in shapes) + 2 * norms
        if self.fp8 or self.int8:
            outs = self.n_heads * d + 2 * self.n_kv_heads * d + h + 2 * self.inter + h
            return mats + (2 if self.fp8 else 4) * outs + 2 * norms
        return itemsize * (mats + norms)


LLAMA_7B = LlamaShape()
LLAMA_70B_FP8 = LlamaShape(n_layers=80, hidden=8192, n_heads=64, n_kv_heads=8, head_dim=128, inter=28672,
                           vocab=32000, max_seq=4096, fp8=True)


class Fp8Linear(nn.Module):
    """y = x @ (W_fp8 * scale[:, None])^T with W in float8_e4m3fn and a bf16 scale per output channel.

    On the GPU (K a multiple of 16) the library's fp8-weight MFMA kernels run:
    a few rows in one launch, up to 64 rows (decode) a split-K kernel or
    64-row tiles, more rows (prefill) a tiled GEMM; all widen the weights to
    bf16 in registers. The decoder groups its q/k/v and gate/up projections into one
    launch each (:func:`fp8_group`). CPU inputs dequantise to bf16 and run a
    bf16 GEMM. Every e4m3 value is exactly
    representable in bf16, so both compute the same products; they differ in
    accumulation order and in rounding the product before the scale.
    """

    def __init__(self, in_features: int, out_features: int) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=torch.float8_e4m3fn),
                                   requires_grad=False)
        self.scale = nn.Parameter(torch.ones(out_features, dtype=torch.bfloat16), requires_grad=False)

    def kernel_eligible(self, x: torch.Tensor) -> bool:
        """Whether the library kernels take this call: a non-empty bf16 GPU input with K a multiple of
        16, and a contiguous, 16-byte aligned weight (``raw_block_transfer`` packs weights back to back
        without alignment; such a weight takes the dequantize path)."""
        k = x.shape[-1]
        m = x.numel() // k if k else 0
        w = self.weight
        return (x.is_cuda and x.dtype == torch.bfloat16 and m > 0 and k % 16 == 0 and m * w.shape[0] < 2**31
                and w.is_contiguous() and w.data_ptr() % 16 == 0)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.kernel_eligible(x):
            k = x.shape[-1]
            y = hip.fp8_linear(x.reshape(x.numel() // k, k), self.weight, self.scale)
            return y.view(*x.shape[:-1], y.shape[-1])
        w = self.weight.to(torch.bfloat16)
        return F.linear(x, w) * self.scale


class _ThroughRounding(torch.autograd.Function):
    """``y`` as it is, with the derivatives that ``x @ (weight * scale[:, None]).T`` has by x."""

    generate_vmap_rule = True

    @staticmethod
    def forward(y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        return y.clone()

    @staticmethod
    def setup_context(ctx, inputs, output) -> None:
        ctx.save_for_backward(*inputs[2:])
        ctx.save_for_forward(*inputs[2:])
        ctx.x_dtype = inputs[1].dtype

    @staticmethod
    def backward(ctx, grad: torch.Tensor):
        weight, scale = ctx.saved_tensors
        return grad, torch.matmul(grad.float() * scale, weight.float()).to(ctx.x_dtype), None, None

    @staticmethod
    def jvp(ctx, dy, dx, dweight, dscale):
        weight, scale = ctx.saved_tensors
        if dx is None:
            return dy
        through = (F.linear(dx.float(), weight.float()) * scale).to(ctx.x_dtype)
        return through if dy is None else dy + through


class Int8Linear(nn.Module):
    """y = x @ (W_int8 * scale[:, None])^T with x rounded to 8 bits, a scale for each row (token).

    On the GPU (bf16 inputs, K a multiple of 16) the library's integer kernels run; the sums of code products are
    exact there. Other calls compute the same codes and their products in float32. Where x needs a gradient it gets
    the one of x @ (W_int8 * scale[:, None])^T: that of the rounding is 0 almost everywhere.
    """

    def __init__(self, in_features: int, out_features: int) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=torch.int8), requires_grad=False)
        self.scale = nn.Parameter(torch.ones(out_features, dtype=torch.float32), requires_grad=False)

    def kernel_eligible(self, x: torch.Tensor) -> bool:
        """Whether the library kernels take this call: non-empty bf16 rows, K a multiple of 16, and a contiguous,
        16-byte aligned weight and scale (``raw_block_transfer`` packs weights back to back without alignment), the
        scale as it was made (``module.bfloat16()`` rounds it)."""
        k = x.shape[-1]
        return (x.numel() > 0 and k % 16 == 0 and k <= hip.INT8_LINEAR_MAX_K and hip.kernel_call(x)
                and self.scale.dtype is torch.float32 and x.numel() // k < 1 << 24
                and hip._packed(self.weight, self.scale)
                and not (self.scale.requires_grad and torch.is_grad_enabled()))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        k = x.shape[-1]
        if self.kernel_eligible(x):
            y = hip.int8_linear(x.reshape(x.numel() // k, k), self.weight, self.scale)
            return y.view(*x.shape[:-1], y.shape[-1])
        xf = x.detach().float()
        scale = xf.abs().amax(-1, keepdim=True) * torch.tensor(1 / INT8_MAX, dtype=torch.float32)
        scale = torch.where(scale < 2.0 ** -100, 0.0, scale)
        codes = (xf * torch.where(scale > 0, 1.0 / scale, 0.0)).round().clamp(-INT8_MAX, INT8_MAX)
        y = (F.linear(codes, self.weight.float()) * scale * self.scale).to(x.dtype)
        if x.requires_grad or torch.autograd.forward_ad._current_level >= 0:
            return _ThroughRounding.apply(y, x, self.weight, self.scale)
        return y


class Int4Linear(nn.Module):
    """y = x @ W^T with W = scale * (code - zero): 4-bit codes, a bf16 scale (and zero, 8 without) for each group of 128
    (64 or 32, as they divide) inputs of a channel, packed as :func:`hip.int4_pack` does.

    On the GPU (bf16 inputs) the library's kernels run. Other calls multiply by the weights in float32, through which x
    gets its gradient.
    """

    def __init__(self, in_features: int, out_features: int, zeros: bool = False) -> None:
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        tiles, units, parts = self._cells(in_features, out_features)
        self.weight = nn.Parameter(torch.empty(tiles, units, 1024, dtype=torch.uint8), requires_grad=False)
        self.scale = nn.Parameter(torch.ones(tiles, units, 16, parts, dtype=torch.bfloat16), requires_grad=False)
        zero = torch.full((tiles, units, 16, parts), 8.0, dtype=torch.bfloat16)
        self.register_parameter("zero", nn.Parameter(zero, requires_grad=False) if zeros else None)

    @staticmethod
    def _cells(in_features: int, out_features: int) -> tuple[int, int, int]:
        """Tiles, units and groups of a unit; the groups are the largest that divide the inputs."""
        group = next((g for g in reversed(hip.INT4_GROUPS) if in_features > 0 and in_features % g == 0), 0)
        if not group:
            raise ValueError(f"4-bit weights have groups of 32 inputs or more, {in_features} are no multiple")
        return -(-out_features // hip.nat.INT4_TILE), -(-in_features // hip.nat.INT4_UNIT), hip.nat.INT4_UNIT // group

    @classmethod
    def nbytes(cls, in_features: int, out_features: int) -> int:
        """Bytes of a layer without zeros."""
        tiles, units, parts = cls._cells(in_features, out_features)
        return tiles * units * (1024 + 2 * 16 * parts)

    @torch.no_grad()
    def quantize_(self, w: torch.Tensor) -> None:
        """Takes weights [out_features, in_features]: the nearest codes under a scale of ``absmax / 7`` for each group, or
        with zeros under ``(max - min) / 15`` and the zero that gives the least weight code 0."""
        if w.shape != (self.out_features, self.in_features):
            raise ValueError(f"weights [{self.out_features}, {self.in_features}] expected, got {tuple(w.shape)}")
        grouped = w.float().unflatten(1, (-1, hip.nat.INT4_UNIT // self.scale.shape[3]))
        zero: torch.Tensor | float = 8.0
        if self.zero is None:
            scale = (grouped.abs().amax(-1) / 7.0).clamp_min(1e-12).to(torch.bfloat16)
        else:
            least = grouped.amin(-1)
            scale = ((grouped.amax(-1) - least) / 15.0).clamp_min(1e-12).to(torch.bfloat16)
            zero = (-least / scale.float()).to(torch.bfloat16)
        shift = zero.float()[..., None] if isinstance(zero, torch.Tensor) else zero
        codes = (grouped / scale.float()[..., None] + shift).round().clamp_(0, 15).flatten(1).to(torch.uint8)
        packed = hip.int4_pack(codes, scale, zero if isinstance(zero, torch.Tensor) else None)
        for held, new in zip((self.weight, self.scale, self.zero), packed):
            if held is not None:
                held.copy_(new)

    def kernel_eligible(self, x: torch.Tensor) -> bool:
        """Whether the library kernels take this call: non-empty bf16 rows, and a contiguous, 16-byte aligned weight, scale
        and zero (``raw_block_transfer`` packs weights back to back without alignment)."""
        held = (self.scale,) if self.zero is None else (self.scale, self.zero)
        k = x.shape[-1]
        return (x.numel() > 0 and k == self.in_features and k <= hip.INT4_MAX_K and hip.kernel_call(x, *held)
                and x.numel() // k < 1 << 24 and hip._packed(self.weight, *held))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.kernel_eligible(x):
            y = hip.int4_linear(x.reshape(-1, self.in_features), self.weight, self.scale, self.zero, self.out_features)
            return y.view(*x.shape[:-1], self.out_features)
        w = hip.int4_dequantize(self.weight, self.scale, self.zero, self.out_features, self.in_features)
        return F.linear(x.float(), w).to(x.dtype)


class Linear(nn.Linear):
    """``nn.Linear`` whose forward on a few bf16 GPU rows (a decode batch) is the library's one-launch kernel."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not torch.jit.is_scripting():  # a scripted module holds torch's operation alone
            if self.bias is None and hip.bf16_linear_eligible(x, self.weight):
                return hip.bf16_linear_unchecked(x, [self.weight])[0]
        return F.linear(x, self.weight, self.bias)


def _plain_call(module: nn.Module) -> bool:
    """Whether calling ``module`` would run its class's forward and nothing else: no forward set on the
    instance (an offload manager's enter/exit trap is one) and no forward hooks. Only then may a caller
    compute the module's output from its weights directly, in a grouped or fused launch."""
    return ("forward" not in module.__dict__ and not module._forward_hooks and not module._forward_pre_hooks
            and not torch_module._global_forward_hooks and not torch_module._global_forward_pre_hooks)


def fp8_group(x: torch.Tensor, layers: list[nn.Module]) -> list[torch.Tensor] | None:
    """The outputs of several ``Fp8Linear`` layers on one input in one grouped kernel launch, or None when
    any of them would not take the kernel, would run more than its own forward when called (an offload
    unit's trap, a hook), or the group's outputs together would reach 2^31 elements, the library's limit
    for one launch (the caller then runs them one by one)."""
    if not all(isinstance(lin, Fp8Linear) and lin.kernel_eligible(x) and _plain_call(lin) for lin in layers):
        return None
    k = x.shape[-1]
    if (x.numel() // k) * sum(lin.weight.shape[0] for lin in layers) >= 2**31:
        return None
    ys = hip.fp8_linear_group(x.reshape(x.numel() // k, k), [lin.weight for lin in layers],
                              [lin.scale for lin in layers])
    return [y.view(*x.shape[:-1], y.shape[-1]) for y in ys]


def int8_group(x: torch.Tensor, layers: list[nn.Module]) -> list[torch.Tensor] | None:
    """The outputs of several ``Int8Linear`` layers on one input, which is rounded to 8 bits once, or None when any of
    them would not take the kernel or would run more than its own forward when called."""
    if not all(isinstance(lin, Int8Linear) and lin.kernel_eligible(x) and _plain_call(lin) for lin in layers):
        return None
    k = x.shape[-1]
    codes, scales = hip.int8_quantize(x.reshape(x.numel() // k, k))
    ys = [hip.int8_matmul(codes, scales, lin.weight, lin.scale) for lin in layers]
    return [y.view(*x.shape[:-1], y.shape[-1]) for y in ys]


def _fusable(x: torch.Tensor, layers: list[nn.Module]) -> bool:
    """Whether a decode-batch call of these ``Fp8Linear`` layers on ``x`` can take a fused epilogue."""
    k = x.shape[-1]
    return (all(isinstance(lin, Fp8Linear) and lin.kernel_eligible(x) and _plain_call(lin) for lin in layers)
            and x.numel() // k <= hip.FP8_DECODE_MAX_ROWS)


def fp8_swiglu(x: torch.Tensor, gate: nn.Module, up: nn.Module) -> torch.Tensor | None:
    """``F.silu(gate(x)) * up(x)`` as one grouped launch whose reduce applies the activation, or None when
    the fused form does not apply (the caller then runs the layers and the activation as usual)."""
    if not _fusable(x, [gate, up]) or gate.weight.shape != up.weight.shape:
        return None
    k = x.shape[-1]
    y = hip.fp8_linear_swiglu(x.reshape(x.numel() // k, k), gate.weight, gate.scale, up.weight, up.scale)
    return y.view(*x.shape[:-1], y.shape[-1])


def fp8_residual(x: torch.Tensor, lin: nn.Module, residual: torch.Tensor) -> torch.Tensor | None:
    """``residual + lin(x)`` with the add folded into the linear's reduce, or None when the fused form
    does not apply (the caller then adds as usual)."""
    if not _fusable(x, [lin]) or residual.dtype != torch.bfloat16 or \
            residual.shape != (*x.shape[:-1], lin.weight.shape[0]):
        return None
    k = x.shape[-1]
    m = x.numel() // k
    y = hip.fp8_linear_residual(x.reshape(m, k), lin.weight, lin.scale, residual.reshape(m, -1))
    return y.view(residual.shape)


def _bf16_fusable(x: torch.Tensor, layers: list[nn.Module]) -> bool:
    """Whether a call of these layers on ``x`` is one launch of the bf16 decode kernel."""
    return (all(type(lin) is Linear and lin.bias is None and _plain_call(lin) for lin in layers)
            and hip.bf16_linear_eligible(x, *[lin.weight for lin in layers]))


def linear_group(x: torch.Tensor, layers: list[nn.Module]) -> list[torch.Tensor] | None:
    """The outputs of several linear layers on one input in one launch, or None when no kernel takes the group."""
    if _bf16_fusable(x, layers):
        return hip.bf16_linear_unchecked(x, [lin.weight for lin in layers])
    if type(layers[0]) is Int8Linear:
        return int8_group(x, layers)
    return fp8_group(x, layers)


def linear_swiglu(x: torch.Tensor, gate: nn.Module, up: nn.Module) -> torch.Tensor | None:
    """``F.silu(gate(x)) * up(x)`` in one launch, or None when no kernel takes the call."""
    if _bf16_fusable(x, [gate, up]) and gate.weight.shape == up.weight.shape:
        return hip.bf16_linear_unchecked(x, [gate.weight, up.weight], hip.nat.FP8_EPILOGUE_SWIGLU)[0]
    return fp8_swiglu(x, gate, up)


def linear_residual(x: torch.Tensor, lin: nn.Module, residual: torch.Tensor) -> torch.Tensor | None:
    """``residual + lin(x)`` in one launch, or None when no kernel takes the call."""
    if _bf16_fusable(x, [lin]) and hip.kernel_call(residual) and residual.is_contiguous() and \
            residual.shape == (*x.shape[:-1], lin.weight.shape[0]):
        return hip.bf16_linear_unchecked(x, [lin.weight], hip.nat.FP8_EPILOGUE_RESIDUAL, residual)[0]
    return fp8_residual(x, lin, residual)


def _proj(s: LlamaShape, n_in: int, n_out: int, dtype: torch.dtype) -> nn.Module:
    if s.int4:
        return Int4Linear(n_in, n_out)
    if s.int8:
        return Int8Linear(n_in, n_out)
    return Fp8Linear(n_in, n_out) if s.fp8 else Linear(n_in, n_out, bias=False, dtype=dtype)


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float, dtype: torch.dtype) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not torch.jit.is_scripting():
            fused = hip.rms_norm(x, self.weight, self.eps)
            if fused is not None:
                return fused
        xf = x.float()
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        return (y * self.weight.float()).to(x.dtype)


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotary embedding with full-width cos/sin tables (halves rotate against each other)."""
    half = x.shape[-1] // 2
    rotated = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * cos + rotated * sin


class Attention(nn.Module):
    def __init__(self, s: LlamaShape, dtype: torch.dtype) -> None:
        super().__init__()
        self.s = s
        self.wq = _proj(s, s.hidden, s.n_heads * s.head_dim, dtype)
        self.wk = _proj(s, s.hidden, s.n_kv_heads * s.head_dim, dtype)
        self.wv = _proj(s, s.hidden, s.n_kv_heads * s.head_dim, dtype)
        self.wo = _proj(s, s.n_heads * s.head_dim, s.hidden, dtype)
        self.q_norm = RMSNorm(s.head_dim, s.eps, dtype) if s.qk_norm else None
        self.k_norm = RMSNorm(s.head_dim, s.eps, dtype) if s.qk_norm else None

    def forward(self, x: torch.Tensor, pos: int, cos: torch.Tensor, sin: torch.Tensor,
                cache_k: torch.Tensor | kv_cache.KVLayer, cache_v: torch.Tensor | None,
                residual: torch.Tensor | None = None) -> torch.Tensor:
        """The attention block's output, plus ``residual`` when given (folded into the output projection's
        launch for decode batches). ``cache_k`` may be a layer of a paged 8-bit cache, which holds both keys and
        values and knows the sequences' positions."""
        s = self.s
        b, t, _ = x.shape
        qkv = linear_group(x, [self.wq, self.wk, self.wv])
        q, k, v = qkv if qkv is not None else (self.wq(x), self.wk(x), self.wv(x))
        q = q.view(b, t, s.n_heads, s.head_dim)
        k = k.view(b, t, s.n_kv_heads, s.head_dim)
        v = v.view(b, t, s.n_kv_heads, s.head_dim)
        norms = {}
        if self.q_norm is not None and self.k_norm is not None:
            # The paged cache's launch normalises too, where calling the norms would run nothing else.
            weights = self.q_norm.weight, self.k_norm.weight
            if (isinstance(cache_k, kv_cache.KVLayer) and _plain_call(self.q_norm) and _plain_call(self.k_norm)
                    and hip.kernel_call(q, *weights) and hip._packed(*weights)):
                norms = {"q_norm": weights[0], "k_norm": weights[1], "eps": s.eps}
            else:
                q, k = self.q_norm(q), self.k_norm(k)
        if isinstance(cache_k, kv_cache.KVLayer):
            o = cache_k.attend(cache_k.append(q, k, v, cos, sin, **norms))
            return self._output(o.view(b, t, s.n_heads * s.head_dim), residual)
        o = hip.rope_attention(q, k, v, cos, sin, pos, cache_k, cache_v)
        if o is not None:
            return self._output(o.view(b, t, s.n_heads * s.head_dim), residual)
        c = cos[pos: pos + t].view(1, t, 1, -1).to(q.dtype)
        sn = sin[pos: pos + t].view(1, t, 1, -1).to(q.dtype)
        q, k = _rotate(q, c, sn), _rotate(k, c, sn)
        cache_k[:b, pos: pos + t] = k
        cache_v[:b, pos: pos + t] = v
        keys = cache_k[:b, : pos + t]
        vals = cache_v[:b, : pos + t]
        rep = s.n_heads // s.n_kv_heads
        if rep > 1:
            keys = keys.repeat_interleave(rep, dim=2)
            vals = vals.repeat_interleave(rep, dim=2)
        qh = q.transpose(1, 2).contiguous()                    # [b, h, t, d]
        kt = keys.permute(0, 2, 3, 1).contiguous()             # [b, h, d, S]  (contiguous right operand)
        vh = vals.transpose(1, 2).contiguous()                 # [b, h, S, d]
        scores = torch.matmul(qh, kt).float() * (1.0 / math.sqrt(s.head_dim))
        if t > 1:
            n = pos + t
            mask = torch.ones(t, n, dtype=torch.bool, device=x.device).triu(diagonal=pos + 1)
            scores = scores.masked_fill(mask, float("-inf"))
        p = torch.softmax(scores, dim=-1).to(vh.dtype)
        o = torch.matmul(p, vh).transpose(1, 2).reshape(b, t, s.n_heads * s.head_dim)
        return self._output(o, residual)

    def _output(self, o: torch.Tensor, residual: torch.Tensor | None) -> torch.Tensor:
        """The output projection of ``o``, plus ``residual`` when given."""
        if residual is None:
            return self.wo(o)
        fused = linear_residual(o, self.wo, residual)
        return fused if fused is not None else residual + self.wo(o)


class DecoderLayer(nn.Module):
    def __init__(self, s: LlamaShape, dtype: torch.dtype) -> None:
        super().__init__()
        self.attn_norm = RMSNorm(s.hidden, s.eps, dtype)
        self.attn = Attention(s, dtype)
        self.mlp_norm = RMSNorm(s.hidden, s.eps, dtype)
        self.gate = _proj(s, s.hidden, s.inter, dtype)
        self.up = _proj(s, s.hidden, s.inter, dtype)
        self.down = _proj(s, s.inter, s.hidden, dtype)

    def forward(self, x: torch.Tensor, pos: int, cos: torch.Tensor, sin: torch.Tensor,
                cache_k: torch.Tensor | kv_cache.KVLayer, cache_v: torch.Tensor | None) -> torch.Tensor:
        x = self.attn(self.attn_norm(x), pos, cos, sin, cache_k, cache_v, residual=x)
        h = self.mlp_norm(x)
        act = linear_swiglu(h, self.gate, self.up)
        if act is None:
            gu = linear_group(h, [self.gate, self.up])
            g, u = gu if gu is not None else (self.gate(h), self.up(h))
            act = hip.silu_mul(g, u)
            if act is None:
                act = F.silu(g) * u
        out = linear_residual(act, self.down, x)
        return out if out is not None else x + self.down(act)


class LlamaModel(nn.Module):
    def __init__(self, s: LlamaShape = LLAMA_7B, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.shape = s
        self.embed = nn.Embedding(s.vocab, s.hidden, dtype=dtype)
        self.layers = nn.ModuleList(DecoderLayer(s, dtype) for _ in range(s.n_layers))
        self.norm = RMSNorm(s.hidden, s.eps, dtype)
        self.lm_head = Linear(s.hidden, s.vocab, bias=False, dtype=dtype)
        inv = 1.0 / (s.rope_theta ** (torch.arange(0, s.head_dim, 2, dtype=torch.float32) / s.head_dim))
        ang = torch.outer(torch.arange(s.max_seq, dtype=torch.float32), inv)
        self.register_buffer("rope_cos", torch.cat([ang.cos(), ang.cos()], -1), persistent=False)
        self.register_buffer("rope_sin", torch.cat([ang.sin(), ang.sin()], -1), persistent=False)
        self.cache_k: list[torch.Tensor] = []
        self.cache_v: list[torch.Tensor] = []

    def init_cache(self, batch: int, max_len: int, device: torch.device) -> None:
        s = self.shape
        shape = (batch, max_len, s.n_kv_heads, s.head_dim)
        dt = self.embed.weight.dtype
        self.cache_k = [torch.zeros(shape, dtype=dt, device=device) for _ in range(s.n_layers)]
        self.cache_v = [torch.zeros(shape, dtype=dt, device=device) for _ in range(s.n_layers)]

    def init_paged_cache(self, pages: int, page_tokens: int = 64, dtype: torch.dtype = torch.float8_e4m3fn,
                         device: torch.device | str = "cuda") -> kv_cache.PagedKVCache:
        """A pool of ``pages`` for this model's layers; its steps go to :meth:`forward`."""
        s = self.shape
        return kv_cache.PagedKVCache(s.n_layers, s.n_kv_heads, s.head_dim, pages, page_tokens, dtype, device)

    def forward(self, tokens: torch.Tensor, pos: int = 0, step: kv_cache.KVStep | kv_cache.KVNodes | None = None,
                every: bool = False) -> torch.Tensor:
        """Logits of the last position, float32. With a ``step`` of a paged cache the tokens are its sequences' next
        ones, or nodes of their trees (``pos`` does not matter), and the logits those of each sequence's last token in the
        step. With ``every`` the logits of all positions, in the weights' type."""
        if step is not None:
            step.check(*tokens.shape, self.rope_cos.shape[0])
        x = self.embed(tokens)
        for i, layer in enumerate(self.layers):
            if step is not None:
                x = layer(x, pos, self.rope_cos, self.rope_sin, step.layer(i), None)
            else:
                x = layer(x, pos, self.rope_cos, self.rope_sin, self.cache_k[i], self.cache_v[i])
        if every:
            return self.lm_head(self.norm(x))
        if step is not None and min(step.counts, default=x.shape[1]) < x.shape[1]:
            last = (step.new.long() - 1).clamp_min(0).view(-1, 1, 1).expand(-1, 1, x.shape[2])
            x = x.gather(1, last)
        return self.lm_head(self.norm(x[:, -1:])).float()


def build_llama(shape: LlamaShape = LLAMA_7B, seed: int = 0, init_device: str = "cpu") -> LlamaModel:
    with torch.device("meta"):
        model = LlamaModel(shape)
    model = model.to_empty(device="cpu")
    s = shape
    inv = 1.0 / (s.rope_theta ** (torch.arange(0, s.head_dim, 2, dtype=torch.float32) / s.head_dim))
    ang = torch.outer(torch.arange(s.max_seq, dtype=torch.float32), inv)
    model.rope_cos.copy_(torch.cat([ang.cos(), ang.cos()], -1))
    model.rope_sin.copy_(torch.cat([ang.sin(), ang.sin()], -1))
    return init_normal_(model, seed, 0.02, init_device)


@torch.no_grad()
def generate(model: LlamaModel, prompt: torch.Tensor, steps: int) -> tuple[torch.Tensor, list[torch.Tensor]]:
    """Greedy decoding with no host synchronisation between steps.

    Returns the generated tokens ``[batch, steps]`` and the logits of every step.
    """
    logits = model(prompt, 0)
    out, all_logits = [], [logits]
    tok = logits.argmax(-1)
    pos = prompt.shape[1]
    for _ in range(steps - 1):
        out.append(tok)
        logits = model(tok, pos)
        all_logits.append(logits)
        tok = logits.argmax(-1)
        pos += 1
    out.append(tok)
    return torch.cat(out, dim=1), all_logits


@torch.no_grad()
def generate_paged(model: LlamaModel, cache: kv_cache.PagedKVCache, prompts: list[list[int]], steps: int,
                   samples: int = 1) -> tuple[list[int], torch.Tensor, list[torch.Tensor]]:
    """Greedy decoding of prompts of different lengths over a paged 8-bit cache.

    The prompts are one ragged pass. Each is then forked into ``samples`` sequences that share its pages; sample j
    starts from its j-th likeliest token. Returns the sequences (in the cache until closed; closed already where an
    error ends the run), their tokens ``[prompts * samples, steps]`` and the logits of every step.
    """
    longest = max(len(p) for p in prompts)
    device = model.rope_cos.device
    tokens = torch.tensor([p + [0] * (longest - len(p)) for p in prompts], device=device)
    roots = [cache.open() for _ in prompts]
    sequences = roots
    try:
        step = cache.begin(roots, [len(p) for p in prompts])
        logits = model(tokens, step=step)
        cache.commit(step)
        sequences = []
        for root in roots:
            sequences += [root, *(cache.fork(root) for _ in range(samples - 1))]
        tok = logits[:, -1].topk(samples, -1).indices.reshape(-1, 1)
        out, all_logits = [tok], [logits]
        for _ in range(steps - 1):
            step = cache.begin(sequences, 1)
            logits = model(tok, step=step)
            cache.commit(step)
            all_logits.append(logits)
            tok = logits.argmax(-1)
            out.append(tok)
    except BaseException:  # the caller has no numbers to close them by
        for s in sequences:
            cache.close(s)
        raise
    return sequences, torch.cat(out, dim=1), all_logits


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`hip.token_logprobs` of logits [..., vocab] and tokens [...]; the results have the tokens' shape, the last two
    with [top] behind it. On the host torch operations."""
    shape, vocab = tokens.shape, logits.shape[-1]
    rows, flat = logits.reshape(-1, vocab), tokens.reshape(-1)
    if rows.is_cuda:
        given, entropy, best, index = hip.token_logprobs(rows, flat, top)
    else:
        logp = torch.log_softmax(rows.float(), -1)
        given = logp.gather(1, flat.clamp(0, vocab - 1)[:, None])[:, 0]
        given = torch.where(flat < 0, 0.0, torch.where(flat < vocab, given, float("nan")))
        entropy = -(logp.exp() * torch.where(logp == float("-inf"), 0.0, logp)).sum(-1)
        index = torch.sort(rows, dim=-1, descending=True, stable=True).indices[:, :top]
        best = logp.gather(1, index)
    return given.view(shape), entropy.view(shape), best.reshape(*shape, top), index.reshape(*shape, top)


@torch.no_grad()
def score(model: LlamaModel, tokens: torch.Tensor, top: int = 0
          ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """What the model makes of tokens [batch, t], as :func:`token_logprobs` returns it for the places [batch, t - 1] behind
    the first: the log probability of the token there, the entropy, and the ``top`` likeliest tokens. Uses the model's own
    cache (:meth:`LlamaModel.init_cache`)."""
    logits = model(tokens, 0, every=True)
    return token_logprobs(logits[:, :-1], tokens[:, 1:], top)


DRAFT_TREE = (-1, 0, 0, 1, 1, 2, 3, 3, 5, 6, 9)  # the likeliest chain of five, and siblings near the root


@torch.no_grad()
def generate_drafted(model: LlamaModel, draft: LlamaModel, cache: kv_cache.PagedKVCache,
                     draft_cache: kv_cache.PagedKVCache, prompts: list[list[int]], steps: int,
                     parents: tuple[int, ...] = DRAFT_TREE) -> tuple[torch.Tensor, torch.Tensor, int]:
    """Greedy decoding over paged 8-bit caches, several tokens for each pass of ``model``: ``draft``, a smaller model of
    the same vocabulary, proposes a tree of tokens behind each sequence, and one pass of ``model`` checks all of its nodes.

    ``parents``: the tree. Node 0 is a sequence's newest token, the others follow level by level; the children of a node
    are the likeliest tokens behind it, in this order. Returns the tokens [prompts, steps], their log probabilities under
    ``model``, and how many passes it made, the prompts' included. Caches and rotary tables need room for a tree's nodes
    beyond the last token; the sequences are closed at the end.
    """
    device = model.rope_cos.device
    n = len(parents)
    if not parents or parents[0] != -1 or -1 in parents[1:]:
        raise ValueError(f"a tree has one root, its first node, got {list(parents)}")
    children = [[c for c, p in enumerate(parents) if p == node] for node in range(n)]
    width = max(map(len, children))
    rank = [children[p].index(c) for c, p in enumerate(parents) if p >= 0]
    before, rank_of = torch.tensor([[-1, *parents[1:]], [0, *rank]], device=device)
    tokens = torch.tensor([p + [0] * (max(map(len, prompts)) - len(p)) for p in prompts], device=device)
    opened: list[tuple[kv_cache.PagedKVCache, int]] = []

    def prompt_pass(m: LlamaModel, c: kv_cache.PagedKVCache) -> tuple[list[int], torch.Tensor]:
        sequences = [c.open() for _ in prompts]
        opened.extend((c, s) for s in sequences)
        step = c.begin(sequences, [len(p) for p in prompts])
        logits = m(tokens, step=step)
        c.commit(step)
        return sequences, logits

    def likeliest(logits: torch.Tensor, top: int) -> tuple[torch.Tensor, torch.Tensor]:
        return token_logprobs(logits, torch.full(logits.shape[:2], -1, device=device), top)[2:]

    try:
        drafted, _ = prompt_pass(draft, draft_cache)
        sequences, logits = prompt_pass(model, cache)
        logp, best = likeliest(logits, 1)
        out, logps = best[:, 0].tolist(), logp[:, 0].tolist()
        passes = 1
        while active := [i for i in range(len(prompts)) if len(out[i]) < steps]:
            nodes = torch.zeros(len(active), n, dtype=torch.int64, device=device)
            nodes[:, 0] = torch.tensor([out[i][-1] for i in active], device=device)
            proposed = draft_cache.draft([drafted[i] for i in active], parents)
            levels = proposed.levels()
            for (lo, hi), (_, end) in zip(levels, [*levels[1:], (n, n)]):  # the last level too: its tokens may be kept
                logits = draft(nodes[:, lo:hi], step=proposed.nodes(lo, hi), every=True)
                if end > hi:
                    _, best = likeliest(logits, width)
                    nodes[:, hi:end] = best[:, before[hi:end] - lo, rank_of[hi:end]]
            checked = cache.draft([sequences[i] for i in active], parents)
            logp, best = likeliest(model(nodes, step=checked.nodes(), every=True), 1)
            passes += 1
            guesses, answers, scores = nodes.tolist(), best[..., 0].tolist(), logp[..., 0].tolist()
            paths = []
            for row, i in enumerate(active):
                path = [0]
                while match := [c for c in children[path[-1]] if guesses[row][c] == answers[row][path[-1]]]:
                    path.append(match[0])
                out[i] += [answers[row][node] for node in path]  # the tokens behind the path's nodes; the last is new
                logps[i] += [scores[row][node] for node in path]
                paths.append(path)
            cache.accept(checked, paths)
            draft_cache.accept(proposed, paths)
    finally:
        for c, s in opened:
            c.close(s)
    return torch.tensor([o[:steps] for o in out]), torch.tensor([x[:steps] for x in logps]), passes


def prompt_tokens(batch: int, length: int, vocab: int, seed: int = 0) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (batch, length), generator=gen)


# ---- Wan-style diffusion transformer -------------------------------------------


@dataclass(frozen=True)
class DiTShape:
    n_blocks: int = 40
    dim: int = 5120
    n_heads: int = 40
    ffn: int = 13824
    eps: float = 1e-6

    @property
    def head_dim(self) -> int:
        return self.dim // self.n_heads

    def block_params(self) -> int:
        d, f = self.dim, self.ffn
        attn = 4 * (d * d + d) + 2 * d  # q, k, v, o with bias + q/k RMSNorm weights
        return 2 * attn + 2 * d + (d * f + f + f * d + d) + 6 * d  # + cross-attn norm, ffn, modulation

    def block_flops(self, tokens: int, text: int) -> float:
        d, f = self.dim, self.ffn
        lin = 2 * tokens * d * d * 4 + 2 * tokens * d * d * 2 + 2 * text * d * d * 2 + 2 * tokens * d * f * 2
        attn = 4 * tokens * tokens * d + 4 * tokens * text * d
        return float(lin + attn)


WAN_DIT = DiTShape()


def sdpa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Attention over [batch, heads, seq, head_dim].

    On the GPU bf16 heads of 64 or 128 values run the library's attention
    kernel; other calls only torch's fused flash / memory-efficient kernels (a
    32760-token score matrix does not belong in HBM, and the unfused path runs
    batched products on transposed views); without a fused kernel this raises.
    """
    if q.device.type == "cuda":
        heads = [t.transpose(1, 2) for t in (q, k, v)] if q.dim() == k.dim() == v.dim() == 4 else None
        if heads is not None and q.shape[1] == k.shape[1] and hip.attention_eligible(*heads):
            return hip.attention_unchecked(*heads).transpose(1, 2)
        from torch.nn.attention import SDPBackend, sdpa_kernel

        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            return F.scaled_dot_product_attention(q, k, v)
    return F.scaled_dot_product_attention(q, k, v)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` whose forward is the library's kernel where it takes the call: the bits of the launch that
    folds the norm into the residual add before it, also where the module is called on its own (as a streamed unit)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not torch.jit.is_scripting():
            fused = hip.residual_norm(x, self.eps, affine=(self.weight, self.bias))
            if fused is not None:
                return fused[1]
        return F.layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)


class _DiTAttention(nn.Module):
    def __init__(self, s: DiTShape, dtype: torch.dtype) -> None:
        super().__init__()
        self.s = s
        self.q = nn.Linear(s.dim, s.dim, dtype=dtype)
        self.k = nn.Linear(s.dim, s.dim, dtype=dtype)
        self.v = nn.Linear(s.dim, s.dim, dtype=dtype)
        self.o = nn.Linear(s.dim, s.dim, dtype=dtype)
        self.norm_q = RMSNorm(s.dim, s.eps, dtype)
        self.norm_k = RMSNorm(s.dim, s.eps, dtype)

    def forward(self, x: torch.Tensor, ctx: torch.Tensor, attn=None) -> torch.Tensor:
        b, n, _ = x.shape
        h, d = self.s.n_heads, self.s.head_dim
        q = self.norm_q(self.q(x)).view(b, n, h, d).transpose(1, 2)
        k = self.norm_k(self.k(ctx)).view(b, ctx.shape[1], h, d).transpose(1, 2)
        v = self.v(ctx).view(b, ctx.shape[1], h, d).transpose(1, 2)
        o = (attn or sdpa)(q, k, v)
        return self.o(o.transpose(1, 2).reshape(b, n, h * d))


class DiTBlock(nn.Module):
    """AdaLN-modulated block: self-attention, cross-attention to text, GELU FFN."""

    def __init__(self, s: DiTShape = WAN_DIT, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.s = s
        self.self_attn = _DiTAttention(s, dtype)
        self.cross_attn = _DiTAttention(s, dtype)
        self.norm3 = LayerNorm(s.dim, eps=s.eps, dtype=dtype)
        self.fc1 = nn.Linear(s.dim, s.ffn, dtype=dtype)
        self.fc2 = nn.Linear(s.ffn, s.dim, dtype=dtype)
        self.modulation = nn.Parameter(torch.zeros(1, 6, s.dim, dtype=dtype))

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        return F.layer_norm(x.float(), (self.s.dim,), eps=self.s.eps).to(x.dtype)

    def _modulate(self, x: torch.Tensor, m: torch.Tensor, scale: int, shift: int) -> torch.Tensor:
        return (self._norm(x).float() * (1 + m[:, scale: scale + 1]) + m[:, shift: shift + 1]).to(x.dtype)

    def forward(self, x: torch.Tensor, e: torch.Tensor, ctx: torch.Tensor, attn=None) -> torch.Tensor:
        """Each residual add and the norm that reads its sum are one launch where the kernel takes the call."""
        adaln = (self.modulation, e)
        eps = self.s.eps

        terms = []

        def m() -> torch.Tensor:  # made once, by the first operation that no kernel takes
            if not terms:
                terms.append(self.modulation.float() + e.float())
            return terms[0]

        fused = hip.residual_norm(x, eps, adaln=adaln, scale=1, shift=0)
        h = fused[1] if fused is not None else self._modulate(x, m(), 1, 0)
        y = self.self_attn(h, h, attn)
        n3 = self.norm3
        plain = type(n3) is LayerNorm and _plain_call(n3)
        fused = hip.residual_norm(x, n3.eps, y, 2, (n3.weight, n3.bias), adaln) if plain else None
        if fused is not None:
            x, h = fused
        else:
            fused = hip.residual_norm(x, eps, y, 2, adaln=adaln)
            x = fused[0] if fused is not None else (x.float() + y.float() * m()[:, 2:3]).to(x.dtype)
            h = n3(x)
        y = self.cross_attn(h, ctx, attn)
        fused = hip.residual_norm(x, eps, y, adaln=adaln, scale=4, shift=3)
        if fused is not None:
            x, h = fused
        else:
            x = x + y
            h = self._modulate(x, m(), 4, 3)
        y = self.fc2(F.gelu(self.fc1(h), approximate="tanh"))
        fused = hip.residual_norm(x, eps, y, 5, adaln=adaln)
        return fused[0] if fused is not None else (x.float() + y.float() * m()[:, 5:6]).to(x.dtype)


class DiTModel(nn.Module):
    def __init__(self, s: DiTShape = WAN_DIT, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.shape = s
        self.blocks = nn.ModuleList(DiTBlock(s, dtype) for _ in range(s.n_blocks))
        self.attn = None  # attention override (callable on [b, h, s, d] tensors)

    def forward(self, x: torch.Tensor, e: torch.Tensor, ctx: torch.Tensor) -> torch.Tensor:
        for blk in self.blocks:
            x = blk(x, e, ctx, self.attn)
        return x


def build_dit(shape: DiTShape = WAN_DIT, seed: int = 0, init_device: str = "cpu") -> DiTModel:
    with torch.device("meta"):
        model = DiTModel(shape)
    model = model.to_empty(device="cpu")
    return init_normal_(model, seed, 0.02, init_device)


def dit_inputs(shape: DiTShape, tokens: int, text: int, seed: int = 0, device: str = "cpu"):
    """Latent tokens, timestep modulation and text context, all ~N(0, 1) in bf16."""
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(1, tokens, shape.dim, generator=gen, device=device).to(torch.bfloat16)
    e = torch.randn(1, 6, shape.dim, generator=gen, device=device).to(torch.bfloat16)
    ctx = torch.randn(1, text, shape.dim, generator=gen, device=device).to(torch.bfloat16)
    return x, e, ctx


# ---- scatter microbenchmark tensor set ------------------------------------------


def scatter_sizes(n: int = 2000, lo: int = 4096, hi: int = 64 << 20, seed: int = 1) -> list[int]:
    """Byte sizes log-uniform in [lo, hi], rounded down to whole bf16 elements."""
    rng = np.random.default_rng(seed)
    u = rng.uniform(math.log(lo), math.log(hi), size=n)
    return [int(math.exp(x)) // 2 * 2 for x in u]


def scatter_shape(nbytes: int, index: int) -> tuple[int, ...]:
    """1-D for even indices, 2-D [rows, cols] (cols = largest power of two <= 1024 dividing numel) for odd."""
    numel = nbytes // 2
    if index % 2 == 0 or numel == 0:
        return (numel,)
    cols = 1
    while cols < 1024 and numel % (cols * 2) == 0:
        cols *= 2
    return (numel // cols, cols)
