"""What the operators between the QKV and the O projection refuse, and their host-only parts, without a GPU: every check is made before
the context is looked at, so a call that passes them all ends at the missing context."""
import ctypes as C
import math
import re

import pytest

from breeze_tts_cpp_b200 import _lib
from breeze_tts_cpp_b200._lib import BF16, F16, F32, FP8, I8, I32, Attention, Cache, RotaryPlan, Tensor

NONE = Tensor(None, 0, 0, 0, 0, -1)
MEMORY = 1 << 40  # addresses that nothing reads


def tensor(at, rows, cols, code=BF16, stride=0, device=0):
    return Tensor(MEMORY + at, rows, cols, stride, code, device)


def cache(pages=4, kv_heads=2, page=16, head_dim=64, code=I8, device=0, at=1 << 30, **other):
    size = pages * kv_heads * page * head_dim
    parts = dict(keys=MEMORY + at, values=MEMORY + at + size, key_scales=MEMORY + at + 2 * size,
                 value_scales=MEMORY + at + 2 * size + size // head_dim * 4)
    parts.update(other)
    return Cache(*(parts[n] for n in ("keys", "values", "key_scales", "value_scales")), pages, kv_heads, page, head_dim, code, device)


def plan(dims=64, scale=1.0, device=0):
    return RotaryPlan(MEMORY + (1 << 29), dims, 0, scale, device)


def refused(name, *arguments):
    """The message; "" when only the context was missing."""
    buffer = C.create_string_buffer(512)
    assert getattr(_lib.load(), name)(None, *(C.byref(a) if isinstance(a, C.Structure) else a for a in arguments), buffer, 512) == -1
    message = buffer.value.decode()
    return "" if "null b200q context" in message else message


def write(c=None, k=None, v=None, slots=None, positions=NONE, rotary=None, q=NONE, q_out=NONE, q_norm=NONE, k_norm=NONE, epsilon=1e-6):
    return refused("b200q_cache_write", c or cache(), k or tensor(0, 3, 128), v or tensor(4096, 3, 128), slots or tensor(8192, 1, 3, I32), positions,
                   rotary, q, q_out, q_norm, k_norm, epsilon)


@pytest.mark.parametrize("other,text", [
    (dict(code=BF16), "INT8 or FP8"), (dict(head_dim=96), "64 or 128"), (dict(page=8), "power of two"), (dict(page=48), "power of two"),
    (dict(page=2048), "power of two"), (dict(pages=0), "empty"), (dict(keys=MEMORY + 8), "16-byte"), (dict(value_scales=None), "16-byte"),
    (dict(pages=1 << 20, kv_heads=64, page=64), "2\\^31"), (dict(values=MEMORY + (1 << 30) + 64), "overlap")])
def test_caches_that_are_none(other, text):
    message = write(cache(**other))
    assert re.search(text, message), message


def test_cache_write_refusals():
    assert write() == ""
    assert write(rotary=plan(), positions=tensor(9000, 1, 3, I32), q=tensor(20000, 3, 256), q_out=tensor(30000, 3, 256), q_norm=tensor(100, 1, 64),
                 k_norm=tensor(400, 1, 64)) == ""
    packed = dict(q=tensor(0, 3, 256, stride=512), k=tensor(512, 3, 128, stride=512), v=tensor(768, 3, 128, stride=512))
    assert write(**packed, q_out=packed["q"]) == ""  # in place in a packed buffer
    assert "overlaps" in write(**packed, q_out=tensor(256, 3, 256, stride=512))  # into the keys' columns
    for call in (dict(k=tensor(0, 3, 128, F32)), dict(v=tensor(4096, 3, 128, F16)), dict(v=tensor(4096, 2, 128)), dict(k=tensor(0, 3, 64))):
        assert "shape/type" in write(**call)
    for call in (dict(slots=tensor(8192, 1, 2, I32)), dict(slots=tensor(8192, 1, 3, F32)), dict(slots=NONE), dict(slots=tensor(8193, 1, 3, I32))):
        assert "slots" in write(**call)
    assert "rotary plan" in write(positions=tensor(9000, 1, 3, I32))
    assert "positions" in write(rotary=plan())
    for bad in (plan(dims=8), plan(dims=24), plan(dims=128), plan(dims=0)):
        assert "multiple of 16" in write(rotary=bad, positions=tensor(9000, 1, 3, I32))
    assert "not finite" in write(rotary=plan(scale=math.inf), positions=tensor(9000, 1, 3, I32))
    assert "another device" in write(rotary=plan(device=1), positions=tensor(9000, 1, 3, I32))
    assert "different devices" in write(k=tensor(0, 3, 128, device=1))
    assert "query" in write(q=tensor(20000, 3, 256))
    assert "query" in write(q=tensor(20000, 3, 96), q_out=tensor(30000, 3, 96))
    assert "without queries" in write(q_norm=tensor(100, 1, 64))
    assert "norm weight" in write(k_norm=tensor(100, 1, 128))
    for epsilon in (-1.0, math.nan, math.inf):
        assert "epsilon" in write(k_norm=tensor(100, 1, 64), epsilon=epsilon)
    assert "overlaps the cache" in write(k=tensor((1 << 30) + 64, 3, 128))


def test_cache_read_refusals():
    def read(slots=None, k=NONE, v=NONE):
        return refused("b200q_cache_read", cache(), slots or tensor(8192, 1, 3, I32), k, v)

    assert read(k=tensor(0, 3, 128)) == "" == read(v=tensor(0, 3, 128, F16))
    assert "no output" in read()
    assert "shape/type" in read(k=tensor(0, 3, 128), v=tensor(4096, 3, 128, F16))
    assert "shape/type" in read(k=tensor(0, 3, 64))
    assert "slots" in read(slots=tensor(8192, 1, 4, I32), k=tensor(0, 3, 128))
    assert "overlap" in read(k=tensor(0, 3, 128), v=tensor(128, 3, 128))
    assert read(k=tensor(0, 3, 128, stride=256), v=tensor(256, 3, 128, stride=256)) == ""  # halves of one buffer
    assert "overlaps" in read(k=tensor(1 << 30, 3, 128))


def test_rotary_refusals():
    def rotary(x=None, positions=None, p=None, head_dim=64, out=None):
        return refused("b200q_rotary", x or tensor(0, 3, 128), positions or tensor(8192, 1, 3, I32), p or plan(), head_dim, out or tensor(4096, 3, 128))

    assert rotary() == "" == rotary(out=tensor(0, 3, 128))
    for call in (dict(x=tensor(0, 3, 128, I8)), dict(out=tensor(4096, 2, 128)), dict(out=tensor(4096, 3, 128, F16))):
        assert "shape/type" in rotary(**call)
    for head_dim in (0, 8, 40, 48, 528):
        assert "fill the row" in rotary(head_dim=head_dim)
    assert "one per row" in rotary(positions=tensor(8192, 1, 2, I32))
    assert "overlaps its input" in rotary(out=tensor(64, 3, 128))
    assert "multiple of 16" in rotary(p=plan(dims=80))
    assert "different devices" in rotary(out=tensor(4096, 3, 128, device=1))


def attention(c=None, **other):
    parts = dict(queries=tensor(0, 3, 256), output=tensor(1 << 20, 3, 256), pages=tensor(1 << 21, 3, 5, I32), lengths=tensor(1 << 22, 1, 3, I32),
                 query_offsets=NONE, prefix_pages=NONE, prefix_length=NONE, scale=0.0)
    parts.update(other)
    return refused("b200q_cached_attention", c or cache(), Attention(*(parts[n] for n, _ in Attention._fields_)))


def test_attention_refusals():
    assert attention() == ""
    assert attention(pages=tensor(1 << 21, 3, 5, I32, stride=9)) == ""
    prefix = dict(prefix_pages=tensor(1 << 23, 1, 4, I32), prefix_length=tensor(1 << 24, 1, 1, I32))
    assert attention(**prefix, query_offsets=tensor(1 << 25, 1, 4, I32)) == ""
    for call in (dict(queries=tensor(0, 3, 256, F32)), dict(output=tensor(1 << 20, 3, 256, F16)), dict(output=tensor(1 << 20, 2, 256))):
        assert "shape/type" in attention(**call)
    assert "multiple of the cache's heads" in attention(queries=tensor(0, 3, 192), output=tensor(1 << 20, 3, 192))
    assert "multiple of the cache's heads" in attention(queries=tensor(0, 3, 200), output=tensor(1 << 20, 3, 200))
    assert "pages" in attention(pages=NONE) and "pages" in attention(pages=tensor(1 << 21, 3, 5, F32))
    assert "lengths" in attention(lengths=tensor(1 << 22, 1, 4, I32))
    assert "one query row" in attention(pages=tensor(1 << 21, 2, 5, I32), lengths=tensor(1 << 22, 1, 2, I32))
    assert "query offsets" in attention(query_offsets=tensor(1 << 25, 1, 3, I32))
    assert "prefix needs" in attention(prefix_pages=prefix["prefix_pages"]) and "prefix needs" in attention(prefix_length=prefix["prefix_length"])
    assert "one int32" in attention(prefix_pages=prefix["prefix_pages"], prefix_length=tensor(1 << 24, 1, 2, I32))
    assert "not finite" in attention(scale=math.nan)
    assert "overlaps" in attention(output=tensor(0, 3, 256)) and "overlaps the cache" in attention(output=tensor(1 << 30, 3, 256))
    assert attention(queries=tensor(0, 3, 256, stride=512), output=tensor(512, 3, 256, stride=512)) == ""
    assert "different devices" in attention(lengths=tensor(1 << 22, 1, 3, I32, device=1))
    large = dict(queries=tensor(0, 1 << 20, 256), output=tensor(1 << 32, 1 << 20, 256), pages=tensor(1 << 34, 2, 1 << 20, I32),
                 lengths=tensor(1 << 22, 1, 2, I32), query_offsets=tensor(1 << 25, 1, 3, I32))
    assert "too many query rows" in attention(cache(at=1 << 36), **large)


def test_addresses_that_no_element_has():
    """Elements lie on multiples of their size; a vector load or store would fault elsewhere."""
    assert "shape/type" in write(k=tensor(1, 3, 128)) and "shape/type" in write(q=tensor(20001, 3, 256), q_out=tensor(30000, 3, 256))
    assert "norm weight" in write(k_norm=tensor(401, 1, 64)) and "slots" in write(slots=tensor(8194, 1, 3, I32))
    assert "misaligned" in write(rotary=RotaryPlan(MEMORY + (1 << 29) + 4, 64, 0, 1.0, 0), positions=tensor(9000, 1, 3, I32))
    assert "shape/type" in attention(queries=tensor(1, 3, 256)) and "shape/type" in attention(output=tensor((1 << 20) + 1, 3, 256))
    assert "pages" in attention(pages=tensor((1 << 21) + 2, 3, 5, I32)) and "lengths" in attention(lengths=tensor((1 << 22) + 1, 1, 3, I32))


def test_tables_whose_last_tile_ends_past_an_int():
    """Positions are counted to the end of a tile of 128 keys in 32 bits."""
    one = dict(queries=tensor(0, 1, 128), output=tensor(1 << 20, 1, 128), lengths=tensor(1 << 22, 1, 1, I32))
    small = cache(kv_heads=1, at=1 << 36)
    most = (2**31 - 128) // 16
    assert attention(small, pages=tensor(1 << 30, 1, most, I32), **one) == ""
    assert "attention pages" in attention(small, pages=tensor(1 << 30, 1, most + 1, I32), **one)
    prefix = dict(pages=tensor(1 << 21, 1, 5, I32), prefix_length=tensor(1 << 24, 1, 1, I32))
    assert attention(small, prefix_pages=tensor(1 << 30, 1, most, I32), **prefix, **one) == ""
    assert "prefix pages" in attention(small, prefix_pages=tensor(1 << 30, 1, most + 1, I32), **prefix, **one)


def test_null_structs_are_errors():
    assert "null cache" in refused("b200q_cache_read", None, tensor(0, 1, 3, I32), tensor(0, 3, 128), NONE)
    assert "null attention" in refused("b200q_cached_attention", cache(), None)
    assert "shape/type" in refused("b200q_rotary", None, None, None, 64, None)


def turns_of(dims, base, scaling="none", factor=1.0, original=0, low=1.0, high=0.0):
    from breeze_tts_cpp_b200 import ops
    plan = ops.Rotary.plan(dims, base, scaling=scaling, factor=factor, original_length=original, low=low, high=high, device="cpu")
    return plan.turns.tolist(), plan.scale


def test_rotary_turns():
    """Against the definitions; powers and logarithms of 64 bits are good to a few units in the last place."""
    dims, base, factor, original = 64, 5e5, 16.0, 4096
    rate = [base ** (-2 * i / dims) / (2 * math.pi) for i in range(dims // 2)]
    close = lambda got, want: all(abs(a - b) <= 1e-14 * b for a, b in zip(got, want)) and len(got) == len(want)  # noqa: E731
    got, scale = turns_of(dims, base)
    assert close(got, rate) and scale == 1
    assert close(turns_of(dims, base, "linear", factor)[0], [r / factor for r in rate])
    stretched = turns_of(dims, base, "base", factor)[0]
    assert abs(stretched[0] - rate[0]) < 1e-15 and abs(stretched[-1] * factor / rate[-1] - 1) < 1e-12  # the fastest kept, the slowest divided
    got, scale = turns_of(dims, base, "wavelength", factor, original, 1.0, 4.0)
    for g, r in zip(got, rate):
        made = original * r
        kept = min(max((made - 1.0) / 3.0, 0.0), 1.0)
        assert abs(g - (r * kept + r / factor * (1 - kept))) <= 1e-14 * r
    assert scale == 1 and got[0] == pytest.approx(rate[0], rel=1e-14) and got[-1] == pytest.approx(rate[-1] / factor, rel=1e-14)
    got, scale = turns_of(dims, base, "yarn", factor, original)
    assert scale == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-6)
    assert got[0] == pytest.approx(rate[0], rel=1e-14) and got[-1] == pytest.approx(rate[-1] / factor, rel=1e-14)
    assert all(r / factor * (1 - 1e-14) <= g <= r * (1 + 1e-14) for g, r in zip(got, rate))
    assert sorted(got, reverse=True) == got


@pytest.mark.parametrize("arguments", [
    dict(dims=0), dict(dims=7), dict(base=1.0), dict(base=math.inf), dict(factor=0.5), dict(factor=math.nan), dict(scaling="yarn"),
    dict(scaling="wavelength", original=4096, low=4.0, high=2.0), dict(scaling="yarn", original=4096, low=0.0), dict(dims=2, scaling="base")])
def test_rotary_turns_refusals(arguments):
    with pytest.raises(_lib.B200QError):
        turns_of(**{"dims": 64, "base": 1e4, **arguments})


def test_unknown_scaling():
    with pytest.raises(ValueError):
        turns_of(64, 1e4, "other")


def test_attention_workspace():
    from breeze_tts_cpp_b200 import ops
    decode = ops.attention_workspace(64, 64, 16, 8, 128)
    assert decode < 8 << 20  # a context's default is enough for decode steps
    assert decode < ops.attention_workspace(64, 64, 16, 8, 128, prefix=True) < ops.attention_workspace(1024, 3, 16, 8, 128, prefix=True)
    for bad in ((1, 0, 16, 8, 128), (1, 1, 16, 3, 128), (1, 1, 16, 8, 96), (-1, 1, 16, 8, 64)):
        with pytest.raises(_lib.B200QError):
            ops.attention_workspace(*bad)


def test_cache_view_checks_its_tensors():
    import torch
    from breeze_tts_cpp_b200 import ops
    view = ops.CacheView.empty(2, 2, 16, 64, FP8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        view.c()
    with pytest.raises(ValueError, match="float64"):
        ops.Rotary(torch.zeros(4)).c()
