"""What the operators of drafted trees, 4-bit weights and token log probabilities refuse, on the host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from flextensor_amd import _native as nat
from flextensor_amd import hip
from flextensor_amd import kv_cache as kvc


def test_operations_refuse_tensors_of_the_host():
    codes, scales = torch.zeros(2, 2, 1, 1, 2048, dtype=torch.int8), torch.zeros(2, 2, 1, 1)
    ints = torch.zeros(1, 1, dtype=torch.int32)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="current GPU"):
        kvc.append(q, q, q, torch.zeros(4, 64), torch.zeros(4, 64), codes, scales, ints, ints[0], q_norm=w, k_norm=w)
    with pytest.raises(ValueError, match="current GPU"):
        kvc.tree_attention(q, codes, scales, ints, ints[0], ints.long())
    with pytest.raises(ValueError, match="current GPU"):
        kvc.keep(codes[None], scales[None], ints, ints[0], ints)
    with pytest.raises(ValueError, match="current GPU"):
        hip.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    packed = hip.int4_pack(torch.zeros(20, 64, dtype=torch.uint8), torch.ones(20, 2).bfloat16())
    with pytest.raises(ValueError, match="current GPU"):
        hip.int4_linear(torch.zeros(1, 64, dtype=torch.bfloat16), *packed)


def test_the_c_entries_refuse_before_they_touch_a_device():
    lib, nul = nat.load(), None
    b = ctypes.c_size_t(7)

    def cache(**change):
        c = nat.Kv8Cache(0, 0, 4, 0, 2, 0, 0, 2, 2, 64, 128, nat.KV8_INT8)
        for k, v in change.items():
            setattr(c, k, v)
        return ctypes.byref(c)

    def append(q_weight=nul, k_weight=nul, eps=1e-5, t=0, at=nul):
        return lib.ftx_kv8_append_norm(cache(), nul, nul, nul, q_weight, k_weight, eps, nul, nul, 8, at, 4, nul, 1, t, 4,
                                       (ctypes.c_int64 * 9)(), nul)

    assert append() == nat.FTX_OK and append(16, 16) == nat.FTX_OK
    for bad in ({"q_weight": 16}, {"k_weight": 16}, {"q_weight": 16, "k_weight": 16, "eps": -1.0},
                {"q_weight": 16, "k_weight": 16, "eps": float("inf")}, {"t": 1}):
        assert append(**bad) == nat.FTX_ERR_INVALID, bad

    def tree(nodes=4, b=1, t=1, tree=nul, stride=1):
        return lib.ftx_kv8_tree_attention(cache(), nul, nul, tree, stride, nodes, b, t, 4, (ctypes.c_int64 * 6)(), 1.0, 100,
                                          nul, 0, nul)

    assert tree(t=0) == tree(b=0) == tree(nodes=64, t=0) == nat.FTX_OK
    for bad in ({"nodes": 65, "t": 0}, {"nodes": -1, "t": 0}, {}, {"tree": 8}):
        assert tree(**bad) == nat.FTX_ERR_INVALID, bad

    def keep(layers=1, b=1, n=1, path=nul, stride=1, **change):
        return lib.ftx_kv8_keep(cache(**change), layers, path, stride, b, n, nul)

    assert keep(layers=0) == keep(b=0) == keep(n=0) == nat.FTX_OK
    for bad in ({"layers": -1}, {"layers": 1 << 20}, {"n": 65}, {"n": -1}, {"b": -1}, {}, {"d": 96}, {"format": 3}):
        assert keep(**bad) in (nat.FTX_ERR_INVALID, nat.FTX_ERR_UNSUPPORTED), bad
    assert lib.ftx_kv8_keep(None, 1, nul, 1, 1, 1, nul) == nat.FTX_ERR_INVALID

    size = lib.ftx_int4_linear_workspace
    for shape, code in (((1, 1, 64, 48), nat.FTX_ERR_UNSUPPORTED), ((1, 1, 65, 64), nat.FTX_ERR_UNSUPPORTED),
                        ((1, 1, (1 << 20) + 128, 128), nat.FTX_ERR_UNSUPPORTED), ((1, 1, 0, 64), nat.FTX_ERR_INVALID),
                        ((-1, 1, 64, 64), nat.FTX_ERR_INVALID), ((1, -1, 64, 64), nat.FTX_ERR_INVALID),
                        ((1 << 40, 2, 64, 64), nat.FTX_ERR_INVALID), ((1 << 30, 1 << 10, 64, 64), nat.FTX_ERR_UNSUPPORTED)):
        assert size(*shape, ctypes.byref(b)) == code, shape
    assert size(0, 64, 64, 32, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert size(1, 64, 64, 32, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert size(64, 128, 8192, 128, ctypes.byref(b)) == nat.FTX_OK and b.value > 0
    assert size(1, 64, 64, 32, None) == nat.FTX_ERR_INVALID

    def linear(m=1, n=16, k=64, stride=64):
        return lib.ftx_int4_linear(nul, stride, nul, nul, nul, nul, m, n, k, 32, nul, 0, nul)

    assert linear(m=0) == linear(n=0) == nat.FTX_OK
    for bad in ({}, {"stride": 32}, {"stride": 68}, {"stride": 1 << 22}):
        assert linear(**bad) == nat.FTX_ERR_INVALID, bad

    size = lib.ftx_token_logprobs_workspace
    for shape in ((1, 0, 0, 0), (-1, 5, 0, 0), (1, 5, 3, 0), (1, 5, 0, 6), (1, 100, 0, 65), (1, 100, 0, -1),
                  (1, 1 << 29, 0, 0), (1 << 40, 1 << 10, 0, 0)):
        assert size(*shape, ctypes.byref(b)) == nat.FTX_ERR_INVALID, shape
    assert size(1 << 30, 100, 0, 0, ctypes.byref(b)) == nat.FTX_ERR_UNSUPPORTED
    assert size(0, 100, 0, 5, ctypes.byref(b)) == size(4096, 32000, 0, 5, ctypes.byref(b)) == nat.FTX_OK and b.value == 0
    assert size(1, 1 << 20, 2, 64, ctypes.byref(b)) == nat.FTX_OK and b.value > 0
    call = lib.ftx_token_logprobs
    assert call(nul, 0, 0, nul, 0, 100, 0, nul, nul, nul, nul, nul, 0, nul) == nat.FTX_OK
    assert call(nul, 100, 0, nul, 1, 100, 0, nul, nul, nul, nul, nul, 0, nul) == nat.FTX_ERR_INVALID
    assert call(16, -1, 0, 16, 2, 100, 0, 16, 16, nul, nul, nul, 0, nul) == nat.FTX_ERR_INVALID


def test_the_torch_binding_leaves_what_it_does_not_know_alone():
    calls = nat.torch_calls()
    t = torch.zeros(2, 2, 2, 64, dtype=torch.bfloat16)
    for name, n in (("append_norm", 16), ("tree_attention", 12), ("keep", 8), ("int4_linear", 7), ("token_logprobs", 5)):
        call = getattr(calls, name)
        for args in ((), (None,) * n, (t,) * (n - 2) + (0, 0), ([],) * (n - 2) + (0, 0)):
            assert call(*args) is None


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (33, 320, 64), (250, 416, 32), (7, 384, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_packed_weights_stand_for_what_was_packed(n, k, group, zeros):
    g = torch.Generator().manual_seed(n + k)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.int64)
    scale = torch.rand(n, k // group, generator=g).bfloat16()
    zero = (16 * torch.rand(n, k // group, generator=g)).bfloat16() if zeros else None
    packed = hip.int4_pack(codes, scale, zero)
    tiles, units = (n + 15) // 16, (k + 127) // 128
    assert packed[0].shape == (tiles, units, 1024) and packed[1].shape == (tiles, units, 16, 128 // group)
    z = zero.float().repeat_interleave(group, 1) if zeros else 8.0
    want = (codes.float() - z) * scale.float().repeat_interleave(group, 1)
    assert torch.equal(hip.int4_dequantize(*packed, n, k), want)
    # the order of the header: lane 16 q + r, word i, input 2 j at bit 4 j, 2 j + 1 at bit 16 + 4 j
    words = packed[0].view(torch.int32).view(tiles, units, 4, 16, 4)
    for ch, at in ((0, 0), (n - 1, k - 1), (n // 2, k // 3)):
        u, rest = divmod(at, 128)
        i, q, e = rest // 32, rest % 32 // 8, rest % 8
        word = int(words[ch // 16, u, q, ch % 16, i])
        assert word >> (4 * (e // 2) + 16 * (e % 2)) & 15 == int(codes[ch, at])


def test_packing_refuses_what_is_no_4_bit_weight():
    codes, scale = torch.zeros(8, 64, dtype=torch.uint8), torch.ones(8, 2).bfloat16()
    for bad in ((codes + 16, scale), (codes.int() - 1, scale), (codes.float(), scale), (codes[0], scale),
                (codes, scale.float()), (codes, scale[:, :1].expand(8, 4)), (codes, scale[:4]), (codes, scale, scale[:, :1]),
                (codes[:, :48], scale)):
        with pytest.raises(ValueError):
            hip.int4_pack(*bad)
