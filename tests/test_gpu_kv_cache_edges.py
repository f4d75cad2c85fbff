"""The 8-bit cache and the int8 linear at the edges of their contracts: scales of zero, infinities, the largest
numbers, gradients that are asked for, memory that runs out. Against float64, and on the types of errors."""

from __future__ import annotations

import math

import pytest
import torch

from flextensor_amd import hip, kv_cache as kvc
from flextensor_amd import workloads as W

pytestmark = pytest.mark.gpu

BLOCK = 32
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FORMATS = list(TOP)


def test_a_layer_whose_scales_were_rounded_runs_in_torch(gpu):
    """``module.bfloat16()`` rounds the channel scales, which the kernels take in fp32."""
    lin = W.init_normal_(W.Int8Linear(64, 32), seed=1).to(gpu).bfloat16()
    x = torch.randn(5, 64, device=gpu, generator=torch.Generator(device=gpu).manual_seed(0)).bfloat16()
    want = lin.cpu()(x.cpu())
    lin = lin.to(gpu)
    assert (lin(x).cpu().float() - want.float()).norm() <= 2.0 ** -8 * want.float().norm()
    assert W.int8_group(x, [lin, lin]) is None


def _inputs(gpu, dtype=torch.int8):
    """q, k, v, cos, sin, codes, scales, table and starts of one sequence of four tokens after three others."""
    g = torch.Generator(device=gpu).manual_seed(1)
    x = [torch.randn(1, 4, h, 64, device=gpu, generator=g).bfloat16() for h in (2, 1, 1)]
    codes = torch.zeros(2, 2, 1, 1, 2048, device=gpu).to(dtype)
    ints = [torch.tensor(v, dtype=torch.int32, device=gpu) for v in ([[0]], [3])]
    return [*x, torch.ones(32, 64, device=gpu), torch.zeros(32, 64, device=gpu), codes, torch.ones(2, 2, 1, 1, device=gpu),
            *ints]


@pytest.mark.parametrize("at", [0, 1, 2, 3, 4, 6])
def test_operands_of_the_cache_that_need_a_gradient_are_refused(gpu, at):
    """q, k, v, cos, sin and the scales; without a gradient the call before and after it is the same."""
    names = ["q", "k", "v", "cos", "sin", "codes", "scales"]
    args = _inputs(gpu)
    args[at].requires_grad_()
    codes = args[5].clone()
    with pytest.raises(ValueError, match=f"append has no backward and {names[at]} "):
        kvc.append(*args)
    assert torch.equal(args[5], codes)  # nothing was written
    if at in (0, 6):
        with pytest.raises(ValueError, match=f"attention has no backward and {names[at]} "):
            kvc.attention(args[0], *args[5:])
    if at == 6:
        with pytest.raises(ValueError, match="copy_pages has no backward and scales "):
            kvc.copy_pages(args[5][None], args[6][None], [0], [1])
    with torch.no_grad():
        got = kvc.append(*args)
        out = kvc.attention(got, *args[5:])
    plain = _inputs(gpu)
    want = kvc.append(*plain)
    assert torch.equal(got, want) and torch.equal(out, kvc.attention(want, *plain[5:]))


def test_scales_of_the_int8_linear_that_need_a_gradient_are_refused(gpu):
    x = torch.randn(3, 64, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)).bfloat16()
    w, scale = torch.ones(8, 64, dtype=torch.int8, device=gpu), torch.ones(8, device=gpu)
    codes, rows = hip.int8_quantize(x)
    trained = scale.clone().requires_grad_()
    with pytest.raises(ValueError, match="int8_linear has no backward and scale "):
        hip.int8_linear(x, w, trained)
    with pytest.raises(ValueError, match="int8_matmul has no backward and scale "):
        hip.int8_matmul(codes, rows, w, trained)
    with pytest.raises(ValueError, match="int8_matmul has no backward and scales "):
        hip.int8_matmul(codes, rows.clone().requires_grad_(), w, scale)
    with torch.no_grad():
        assert torch.equal(hip.int8_linear(x, w, trained), hip.int8_linear(x, w, scale))
    # the module's own scale: its gradient, in torch
    lin = W.init_normal_(W.Int8Linear(64, 8), seed=3).to(gpu)
    lin.scale.requires_grad_()
    lin(x).float().sum().backward()
    assert lin.scale.grad.isfinite().all() and lin.scale.grad.any()


def test_memory_that_runs_out_is_torchs_own_error(gpu):
    """A result of 1 GiB where 64 MiB are left: no kernel has started when it is asked for."""
    q = torch.zeros(1, 1 << 17, 64, 64, dtype=torch.bfloat16, device=gpu)
    codes, scales = torch.zeros(1, 2, 1, 1, 2048, dtype=torch.int8, device=gpu), torch.zeros(1, 2, 1, 1, device=gpu)
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    cos = torch.zeros(32, 64, device=gpu)
    x, w = torch.zeros(1 << 13, 64, dtype=torch.bfloat16, device=gpu), torch.zeros(1 << 16, 64, dtype=torch.int8, device=gpu)
    scale = torch.ones(1 << 16, device=gpu)
    rows, row_scales = hip.int8_quantize(x)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(gpu).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved(gpu) + (64 << 20)) / total)
    try:
        for call in (lambda: kvc.attention(q, codes, scales, table, table[0]),
                     lambda: kvc.append(q, q[:, :, :1], q[:, :, :1], cos, cos, codes, scales, table, table[0]),
                     lambda: hip.int8_linear(x, w, scale), lambda: hip.int8_matmul(rows, row_scales, w, scale)):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("small", [0.0, 1e-36])
def test_infinities_among_zeros_are_stored_as_zeros(gpu, dtype, small):
    """A block whose finite values make no scale: all of its codes are 0 but those of NaN; what is appended to it
    later has a scale of its own, and attention sees zeros."""
    kv, d = 2, 64
    codes, scales = torch.zeros(2, 2, kv, 1, BLOCK * d, device=gpu).to(dtype), torch.ones(2, 2, kv, 1, device=gpu)
    table = torch.tensor([[1]], dtype=torch.int32, device=gpu)
    cos, sin = torch.ones(BLOCK, d, device=gpu), torch.zeros(BLOCK, d, device=gpu)
    q = torch.ones(1, 5, 2, d, dtype=torch.bfloat16, device=gpu)
    k, v = (torch.full((1, 5, kv, d), small, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    v[0, 1, 0, 3], v[0, 2, 0, 40], v[0, 4, 1, 7] = float("inf"), float("-inf"), float("nan")
    starts = torch.tensor([0], dtype=torch.int32, device=gpu)
    kvc.append(q, k, v, cos, sin, codes, scales, table, starts)
    assert not scales[1].any()
    keys, values = kvc.read(codes, scales, table[0])
    nan = torch.zeros(BLOCK, kv, d, dtype=torch.bool, device=gpu)
    nan[4, 1, 7] = dtype != torch.int8
    assert not keys.any() and torch.equal(values.isnan(), nan) and not values.nan_to_num(0.0).any()
    out = kvc.attention(q, codes, scales, table, starts)
    assert torch.equal(out[0, 4].isnan(), nan[4]) and not out[0].isnan()[:, ~nan[4]].any()
    assert not out.nan_to_num(0.0).any()
    # three more tokens, of ones: the scale that they make, the infinities' codes still 0
    one = torch.ones(1, 3, kv, d, dtype=torch.bfloat16, device=gpu)
    kvc.append(one, one, one, cos, sin, codes, scales, table, starts + 5)
    keys, values = kvc.read(codes, scales, table[0])
    want = torch.zeros(BLOCK, kv, d, device=gpu)
    want[5:8] = TOP[dtype] * (torch.ones((), device=gpu) * (1 / TOP[dtype]))
    assert torch.equal(keys, want) and torch.equal(values.nan_to_num(0.0), want)


def _pool(gpu, pages, kv, page, d, dtype, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + pages)
    top = TOP[dtype]
    y = torch.randn(pages, 2, kv, page // BLOCK, BLOCK * d, device=gpu, generator=g).mul_(top / 4).clamp_(-top, top)
    return (y.round() if dtype == torch.int8 else y).to(dtype), \
        torch.exp(0.3 * torch.randn(y.shape[:-1], device=gpu, generator=g)) * (4 / top)


def _attend64(q, codes, scales, table, start):
    """One sequence in float64, head by head over what :func:`kvc.read` says that the codes stand for."""
    _, t, h, d = q.shape
    kv = codes.shape[2]
    keys, values = (x[0, : start + t].double() for x in kvc.read(codes, scales, table))
    seen = torch.arange(start + t, device=q.device) <= start + torch.arange(t, device=q.device)[:, None]
    out = torch.zeros(1, t, h, d, dtype=torch.float64, device=q.device)
    for head in range(h):
        k, v = (x[:, head // (h // kv)].contiguous() for x in (keys, values))
        s = (q[0, :, head].double() @ k.t().contiguous() / math.sqrt(d)).masked_fill(~seen, -math.inf)
        out[0, :, head] = torch.softmax(s, -1) @ v
    return out


# tokens, heads, kv heads, d, page, start: a row, a tile of 16 rows over split keys, tiles of 32, tiles of 256 unsplit and
# split
SHAPES = [(1, 2, 2, 64, 32, 100), (1, 8, 1, 128, 64, 9000), (20, 4, 2, 64, 32, 70), (300, 64, 64, 128, 64, 0),
          (64, 64, 8, 64, 64, 30000)]
TWO_ROUNDINGS = 2.0 ** -7  # of the probabilities (2^-8 of each at most, less in a sum of many) and of the output


def _case(gpu, dtype, t, h, kv, d, page, start):
    pages = -(-(start + t) // page)
    codes, scales = _pool(gpu, pages, kv, page, d, dtype)
    g = torch.Generator(device=gpu).manual_seed(t + h)
    table = torch.randperm(pages, device=gpu, generator=g).view(1, pages).int()
    q = torch.randn(1, t, h, d, device=gpu, generator=g).mul(2.0).bfloat16()
    return q, codes, scales, table, torch.tensor([start], dtype=torch.int32, device=gpu)


def _check(got, want):
    got = got.double()
    assert got.isfinite().all()
    assert (got - want).norm() <= TWO_ROUNDINGS * want.norm()
    assert ((got - want).norm(dim=-1) <= 4 * TWO_ROUNDINGS * want.norm(dim=-1)).all()


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -101])
def test_blocks_without_a_scale_stand_for_zeros(gpu, dtype, shape, scale):
    """Their codes, which are none of them 0, weigh in the sum and add nothing: the first and every third block."""
    q, codes, scales, table, starts = _case(gpu, dtype, *shape)
    start = shape[-1]
    for block in range(0, table.shape[1] * codes.shape[3], 3):
        scales[int(table[0, block // codes.shape[3]]), 1, :, block % codes.shape[3]] = scale
    want = _attend64(q, codes, scales, table, start)
    if start == 0:  # the first tokens see the first block alone
        assert not kvc.attention(q, codes, scales, table, starts)[0, :BLOCK].float().abs().gt(1e-25).any()
        got = kvc.attention(q, codes, scales, table, starts)[:, BLOCK:]
        _check(got, want[:, BLOCK:])
        return
    _check(kvc.attention(q, codes, scales, table, starts), want)


def test_a_nan_code_without_a_scale_is_a_nan(gpu):
    """c * 0 of a NaN."""
    q, codes, scales, table, starts = _case(gpu, torch.float8_e4m3fn, 1, 2, 2, 64, 32, 100)
    page = int(table[0, 1])
    scales[page, 1] = 0.0
    codes.view(torch.uint8)[page, 1, 1, 0, 5 * BLOCK + 9] = 0x7F
    out = kvc.attention(q, codes, scales, table, starts)
    nan = torch.zeros(1, 1, 2, 64, dtype=torch.bool, device=gpu)
    nan[0, 0, 1, 5] = True
    assert torch.equal(out.isnan(), nan)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("near", ["large", "small", "both"])
def test_values_over_the_range_that_the_sums_hold(gpu, dtype, shape, near):
    """Values of up to 2^100, and down to the smallest scale, alone and in turn by block."""
    q, codes, scales, table, starts = _case(gpu, dtype, *shape)
    start = shape[-1]
    spread = scales[:, 1].clamp(max=4 / TOP[dtype]) * (TOP[dtype] / 4)  # exp(0.3 n), 1 at most
    scales[:, 1] = (spread * 2.0 ** -99).clamp(min=2.0 ** -100) if near == "small" else spread * (2.0 ** 100 / TOP[dtype])
    if near == "both":
        for block in range(1, table.shape[1] * codes.shape[3], 2):
            scales[int(table[0, block // codes.shape[3]]), 1, :, block % codes.shape[3]] = 2.0 ** -99
    _check(kvc.attention(q, codes, scales, table, starts), _attend64(q, codes, scales, table, start))


def test_more_long_rows_than_a_launch_of_wide_workgroups_holds(gpu):
    """2^22 rows of 8208 values: 2^32 threads would be one too many where a row has 1024."""
    m, k = 1 << 22, 8208
    need = m * (2 * k + 8448 + 4)
    if torch.cuda.mem_get_info(gpu)[0] + torch.cuda.memory_reserved(gpu) - torch.cuda.memory_allocated(gpu) < need + (8 << 30):
        pytest.skip(f"needs {need >> 30} GiB")
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=gpu)
    rows = [0, 1, m // 2 + 5, m - 1]
    some = torch.randn(4, k, device=gpu, generator=torch.Generator(device=gpu).manual_seed(0)).bfloat16()
    x[rows] = some
    try:
        codes, scales = hip.int8_quantize(x)
        want, want_scales = hip.int8_quantize(some)
        assert torch.equal(codes[rows], want) and torch.equal(scales[rows], want_scales)
        assert not scales[2: m // 2].any() and not codes[m // 2 + 6: m // 2 + 5000].any()
    finally:
        del x
        codes = None
        torch.cuda.empty_cache()


@pytest.mark.parametrize("int8", [False, True])
def test_a_decoder_step_of_no_sequences(gpu, int8):
    shape = W.LlamaShape(n_layers=2, hidden=128, n_heads=2, n_kv_heads=1, head_dim=64, inter=192, vocab=50, max_seq=64,
                         int8=int8)
    model = W.build_llama(shape, seed=0).to(gpu)
    cache = model.init_paged_cache(4, 32, torch.int8, gpu)
    step = cache.begin([], [], tokens=2)
    with torch.no_grad():
        assert model(torch.zeros(0, 2, dtype=torch.long, device=gpu), step=step).shape == (0, 1, 50)
    cache.commit(step)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row(gpu, shape, value):
    """An infinity gives scores of both infinities or NaN: no softmax of them is a number."""
    q, codes, scales, table, starts = _case(gpu, torch.int8, *shape)
    want = _attend64(q, codes, scales, table, shape[-1])
    t, h = shape[:2]
    bad = torch.zeros(1, t, h, dtype=torch.bool, device=gpu)
    bad[0, t // 2, h - 1] = bad[0, t - 1, 0] = True
    q[bad] = torch.where(torch.arange(q.shape[3], device=gpu) % 17 == 3, value, q[bad])
    got = kvc.attention(q, codes, scales, table, starts)
    assert got[bad].isnan().all()
    if not bad.all():
        _check(got[~bad], want[~bad])


@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_that_is_not_a_number_spoils_the_rows_that_see_it(gpu, shape):
    """An e4m3 NaN among a head's keys: rows from its token on, of the queries that share the head."""
    q, codes, scales, table, starts = _case(gpu, torch.float8_e4m3fn, *shape)
    t, h, kv, d, page, start = shape
    want = _attend64(q, codes, scales, table, start)
    at = start + t // 2
    cell = codes.view(torch.uint8)[int(table[0, at // page]), 0, kv - 1, at % page // BLOCK]
    cell.view(d // 16, BLOCK, 16)[1, at % BLOCK, 5] = 0x7F
    got = kvc.attention(q, codes, scales, table, starts)
    bad = torch.zeros(1, t, h, dtype=torch.bool, device=gpu)
    bad[0, t // 2:, (kv - 1) * (h // kv):] = True
    assert got[bad].isnan().all()
    if not bad.all():
        _check(got[~bad], want[~bad])


def test_a_decoder_ends_at_its_last_position_on_pages_used_before(gpu):
    """Every page holds NaN codes of an earlier sequence. Up to the last position the logits are numbers; a step past it
    is refused, writes nothing and counts nothing."""
    shape = W.LlamaShape(n_layers=2, hidden=128, n_heads=2, n_kv_heads=1, head_dim=64, inter=192, vocab=50, max_seq=40)
    model = W.build_llama(shape, seed=0).to(gpu)
    cache = model.init_paged_cache(4, 32, torch.float8_e4m3fn, gpu)
    cache.codes.view(torch.uint8).fill_(0x7F)
    cache.scales.fill_(1.0)
    seq = cache.open()
    with torch.no_grad():
        for n in (37, 3):
            step = cache.begin([seq], n)
            assert model(torch.ones(1, n, dtype=torch.long, device=gpu), step=step).isfinite().all()
            cache.commit(step)
        before = cache.codes.view(torch.uint8).clone(), cache.scales.clone()
        step = cache.begin([seq], 1)
        with pytest.raises(ValueError, match="40 positions"):
            model(torch.ones(1, 1, dtype=torch.long, device=gpu), step=step)
    assert torch.equal(cache.codes.view(torch.uint8), before[0]) and torch.equal(cache.scales, before[1])
    assert cache.length(seq) == 40
