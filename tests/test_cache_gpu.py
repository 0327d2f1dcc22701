"""Rotary positions and the quantized key/value cache against their 64-bit forms."""
import pytest
import torch

from breeze_tts_cpp_b200 import _lib, ops
from tests.cache_reference import F32_HALF, RANGE, half_step, held, least, normed, turned

pytestmark = pytest.mark.gpu
FORMATS = {"int8": ops.I8, "fp8": ops.FP8}
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def normal(seed, *shape, dtype=torch.bfloat16, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def plan(dims, interleaved=False, scaling="none"):
    return ops.Rotary.plan(dims, 1e6, interleaved, scaling, factor=8.0 if scaling != "none" else 1.0, original_length=8192)


def rotary_bound(x, want, dtype, scale):
    """Half a step of the result; an angle good to 2^-24 turns, cosine and sine to two half steps, two products and a sum."""
    reach = x.abs().amax(-1, keepdim=True) * scale
    return want.abs() * half_step(dtype) + least(dtype) + reach * 2 * (6.3 + 2 + 3) * F32_HALF


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,head_dim,dims,scaling", [(1, 1, 16, 16, "none"), (3, 16, 64, 32, "linear"), (65, 5, 128, 128, "yarn"),
                                                              (7, 3, 80, 48, "base"), (2, 40, 128, 96, "wavelength"), (5, 2, 512, 512, "none")])
def test_rotary(ctx_factory, rows, heads, head_dim, dims, scaling, interleaved, dtype):
    ctx, dtype = ctx_factory("int8"), DTYPES[dtype]
    rotary = plan(dims, interleaved, scaling)
    x = normal(rows, rows, heads * head_dim, dtype=dtype)
    positions = torch.arange(rows, dtype=torch.int32) * 40007 - 11
    want = turned(x.double().view(rows, heads, head_dim), positions, rotary.turns.cpu(), interleaved, rotary.scale)
    bound = rotary_bound(x.double().view(rows, heads, head_dim), want, dtype, rotary.scale)
    out = ctx.rotary(x.cuda(), positions.cuda(), rotary, head_dim)
    torch.cuda.synchronize()
    assert ((out.cpu().double().view(want.shape) - want).abs() <= bound).all()
    assert torch.equal(out.cpu().view(rows, heads, head_dim)[..., dims:], x.view(rows, heads, head_dim)[..., dims:])
    # in place, on a slice of a packed buffer that begins at an odd element
    packed = torch.zeros(rows, heads * head_dim + 9, dtype=dtype, device="cuda")
    part = packed[:, 3: 3 + heads * head_dim]
    part.copy_(x)
    ctx.rotary(part, positions.cuda(), rotary, head_dim, out=part)
    torch.cuda.synchronize()
    assert torch.equal(part, out) and not packed[:, :3].any() and not packed[:, 3 + heads * head_dim:].any()


def test_rotary_far_positions_keep_their_angles(ctx_factory):
    ctx, rotary = ctx_factory("int8"), plan(128)
    positions = torch.tensor([2**31 - 1, -(2**31), 10**9 + 7, 131071], dtype=torch.int32)
    x = normal(1, 4, 128, dtype=torch.float16)
    want = turned(x.double().view(4, 1, 128), positions, rotary.turns.cpu(), False, 1.0)
    out = ctx.rotary(x.cuda(), positions.cuda(), rotary, 128).cpu().double().view(4, 1, 128)
    # 2^31 turns take 31 of the product's 53 bits; the remainder is good to 2^-22, both sides.
    bound = rotary_bound(x.double().view(4, 1, 128), want, torch.float16, 1.0) + x.double().abs().max() * 2 * 6.3 * 2.0**-22
    assert ((out - want).abs() <= bound).all()


def check_stored(cache, fmt, slots, want, which, loose):
    """Every byte is the nearest one of its row, but for a value within `loose` of a border; slots out of range wrote nothing."""
    values, scales = (cache.keys, cache.key_scales) if which == "k" else (cache.values, cache.value_scales)
    values, scales = held(values.cpu(), fmt), scales.cpu().double()
    page = values.shape[2]
    for r, slot in enumerate(slots.tolist()):
        if not 0 <= slot < values.shape[0] * page:
            continue
        got, scale = values[slot // page, :, slot % page], scales[slot // page, :, slot % page, None]
        x = want[r]
        most = x.abs().amax(-1, keepdim=True)
        right = torch.where(most == 0, torch.ones_like(most), most / RANGE[fmt])
        assert ((scale - right).abs() <= right * loose).all()
        part = x / right
        step = torch.full_like(part, 0.5) if fmt == ops.I8 else torch.maximum(part.abs() * half_step(torch.float8_e4m3fn), torch.tensor(2.0**-10))
        assert ((got - part).abs() <= step * (1 + 2 * loose) + part.abs() * loose).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,heads,kv_heads,head_dim,page,interleaved,norm", [
    (1, 1, 1, 64, 16, False, True), (5, 16, 8, 128, 64, False, True), (67, 6, 3, 64, 32, True, False), (9, 24, 8, 128, 1024, True, True),
    (33, 5, 5, 128, 16, False, False), (4, 40, 4, 64, 128, False, True)])
def test_cache_write(ctx_factory, rows, heads, kv_heads, head_dim, page, interleaved, norm, fmt, dtype):
    ctx, dtype, fmt = ctx_factory("int8"), DTYPES[dtype], FORMATS[fmt]
    rotary = plan(head_dim // 2 if rows % 2 else head_dim, interleaved, "yarn")
    packed = normal(rows, rows, (heads + 2 * kv_heads) * head_dim, dtype=dtype).cuda()
    packed[0, heads * head_dim: (heads + 1) * head_dim] = 0  # a key of zeros
    q, k, v = packed.split((heads * head_dim, kv_heads * head_dim, kv_heads * head_dim), 1)
    cache = ops.CacheView.empty(-(-rows // page) + 2, kv_heads, page, head_dim, fmt)
    for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
        t.fill_(7)
    total = cache.keys.shape[0] * page
    slots = torch.randperm(total, generator=torch.Generator().manual_seed(rows))[:rows].to(torch.int32)
    if rows > 4:
        slots[1], slots[3] = -1, total
    positions = torch.arange(rows, dtype=torch.int32) * 977 + 5
    weights = [normal(3 + i, head_dim, dtype=dtype, std=0.2, mean=1.0) if norm else None for i in range(2)]
    q_out = torch.empty(rows, heads * head_dim, dtype=dtype, device="cuda")
    on = [w.cuda() if norm else None for w in weights]
    ctx.cache_write(cache, k, v, slots.cuda(), positions.cuda(), rotary, q, q_out, *on, epsilon=1e-5)
    torch.cuda.synchronize()
    heads_of = lambda x: x.cpu().double().view(rows, -1, head_dim)  # noqa: E731
    turn = lambda x: turned(x, positions, rotary.turns.cpu(), interleaved, rotary.scale)  # noqa: E731
    want_q, want_k = (turn(normed(heads_of(x), w, 1e-5)) for x, w in zip((q, k), weights))
    # A sum of up to 128 squares (relative 7 halvings + 4 serial terms of a lane), a root, a quotient and two products, then the rotation.
    loose = (24 + 23) * F32_HALF * 2
    reach = want_q.abs().amax(-1, keepdim=True)
    assert ((heads_of(q_out) - want_q).abs() <= want_q.abs() * half_step(dtype) + least(dtype) + reach * 2 * loose).all()
    check_stored(cache, fmt, slots, want_k, "k", 4 * loose)
    check_stored(cache, fmt, slots, heads_of(v), "v", 3 * F32_HALF * 2)
    untouched = torch.ones(total, dtype=torch.bool)
    untouched[slots[(slots >= 0) & (slots < total)].long()] = False
    for t in (cache.keys, cache.values):
        assert (t.cpu().transpose(1, 2).flatten(0, 1)[untouched] == 7).all()
    for t in (cache.key_scales, cache.value_scales):
        assert (t.cpu().transpose(1, 2).flatten(0, 1)[untouched] == 7).all()
    # the same in place: queries keep their place in the packed buffer
    again = packed.clone()
    q2, k2, v2 = again.split((heads * head_dim, kv_heads * head_dim, kv_heads * head_dim), 1)
    ctx.cache_write(cache, k2, v2, slots.cuda(), positions.cuda(), rotary, q2, q2, *on, epsilon=1e-5)
    torch.cuda.synchronize()
    assert torch.equal(q2, q_out) and torch.equal(again[:, heads * head_dim:], packed[:, heads * head_dim:])


@pytest.mark.parametrize("fmt", FORMATS)
def test_cache_write_without_positions_is_the_row_quantizer(ctx_factory, fmt):
    ctx, fmt, rows, kv_heads, head_dim, page = ctx_factory("int8"), FORMATS[fmt], 21, 3, 128, 16
    k, v = (normal(i, rows, kv_heads * head_dim, std=3.0).cuda() for i in range(2))
    cache = ops.CacheView.empty(2, kv_heads, page, head_dim, fmt)
    slots = torch.arange(rows, dtype=torch.int32, device="cuda")
    ctx.cache_write(cache, k, v, slots)
    for x, values, scales in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
        rows_of = ctx.quantize_rows(x.view(rows * kv_heads, head_dim), ops.RowScaledView.empty(rows * kv_heads, head_dim, fmt))
        torch.cuda.synchronize()
        assert torch.equal(values.transpose(1, 2).flatten(0, 1)[:rows].reshape(rows * kv_heads, head_dim), rows_of.values)
        assert torch.equal(scales.transpose(1, 2).flatten(0, 1)[:rows].reshape(-1), rows_of.scales.view(-1))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_are_not_finite_read_back_as_nan(ctx_factory, fmt):
    ctx, fmt = ctx_factory("int8"), FORMATS[fmt]
    x = normal(5, 4, 2 * 64).cuda()
    x[1, 3], x[2, 70], x[3, 127] = float("nan"), float("inf"), -float("inf")
    cache = ops.CacheView.empty(1, 2, 16, 64, fmt)
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    ctx.cache_write(cache, x, x, slots)
    k, v = torch.empty_like(x), torch.empty_like(x)
    ctx.cache_read(cache, slots, k, v)
    torch.cuda.synchronize()
    bad = torch.tensor([[False, False], [True, False], [False, True], [False, True]])
    for y in (k, v):
        assert torch.equal(torch.isnan(y).view(4, 2, 64).all(-1).cpu(), bad) and torch.equal(torch.isnan(y).view(4, 2, 64).any(-1).cpu(), bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,kv_heads,head_dim,page", [(1, 1, 64, 16), (37, 3, 128, 32), (70, 8, 64, 16), (300, 40, 128, 64)])
def test_cache_read(ctx_factory, rows, kv_heads, head_dim, page, fmt, dtype):
    ctx, dtype, fmt, pages = ctx_factory("int8"), DTYPES[dtype], FORMATS[fmt], 3
    g = torch.Generator().manual_seed(rows)
    values = [torch.randint(0, 256, (pages, kv_heads, page, head_dim), generator=g, dtype=torch.uint8) for _ in range(2)]
    if fmt == ops.FP8:
        for x in values:
            x[(x & 0x7f) == 0x7f] = 0x7e
    scales = [torch.rand(pages, kv_heads, page, generator=g) for _ in range(2)]
    cache = ops.CacheView(*(x.cuda() for x in values), *(x.cuda() for x in scales), fmt)
    slots = torch.randint(-2, pages * page + 2, (rows,), generator=g, dtype=torch.int32)
    slots[0] = pages * page - 1
    packed = torch.full((rows, 2 * kv_heads * head_dim + 5), 3.0, dtype=dtype, device="cuda")
    k, v = packed[:, 1: 1 + kv_heads * head_dim], packed[:, 1 + kv_heads * head_dim: 1 + 2 * kv_heads * head_dim]
    ctx.cache_read(cache, slots.cuda(), k, v)
    alone = torch.empty(rows, kv_heads * head_dim, dtype=dtype, device="cuda")
    ctx.cache_read(cache, slots.cuda(), None, alone)
    torch.cuda.synchronize()
    inside = (slots >= 0) & (slots < pages * page)
    for got, x, s in ((k, values[0], scales[0]), (v, values[1], scales[1]), (alone, values[1], scales[1])):
        rows_of = (held(x, fmt).float() * s[..., None]).transpose(1, 2).flatten(0, 1).flatten(1)
        want = torch.where(inside[:, None], rows_of[slots.clamp(0, pages * page - 1).long()], torch.zeros(())).to(dtype)
        assert torch.equal(got.cpu(), want)
    assert (packed[:, 0] == 3).all() and (packed[:, 1 + 2 * kv_heads * head_dim:] == 3).all()


def test_refusals_reach_the_caller(ctx_factory):
    ctx = ctx_factory("int8")
    cache = ops.CacheView.empty(2, 2, 16, 64, ops.I8)
    x, slots = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for call, text in ((lambda: ctx.cache_write(cache, x, x.half(), slots), "type mismatch"),
                       (lambda: ctx.cache_write(cache, x, x, slots.float()), "int32"),
                       (lambda: ctx.cache_write(cache, x, x, slots[:2]), "one per row"),
                       (lambda: ctx.cache_write(cache, x, x, slots, positions=slots), "rotary plan"),
                       (lambda: ctx.cache_read(cache, slots, None, None), "no output"),
                       (lambda: ctx.rotary(x, slots, plan(128), 64), "multiple of 16"),
                       (lambda: ctx.rotary(x, slots, plan(64), 48), "fill the row")):
        with pytest.raises(_lib.B200QError, match=text):
            call()
    with pytest.raises(ValueError, match="contiguous"):
        ctx.cache_read(ops.CacheView(cache.keys.cpu(), *cache_parts(cache)[1:], ops.I8), slots, x, x)


def cache_parts(cache):
    return cache.keys, cache.values, cache.key_scales, cache.value_scales
