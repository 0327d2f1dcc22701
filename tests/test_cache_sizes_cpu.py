"""What the cache operators refuse, beyond test_cache_cpu.py, without a GPU: sizes past 32 or 64 bits, outputs over the rotary plan."""
import pytest

from breeze_tts_cpp_b200._lib import I32, Cache, Tensor
from tests.test_cache_cpu import MEMORY, NONE, refused, tensor


def cache(pages, kv_heads, page=16, head_dim=64):
    """Storage 2^44 bytes apart: no overlap, whatever the sizes."""
    return Cache(*(MEMORY + (i << 44) for i in range(1, 5)), pages, kv_heads, page, head_dim, 4, 0)


def empty(rows, cols=0):
    return Tensor(MEMORY, rows, cols, 0, 0, 0)


@pytest.mark.parametrize("pages,kv_heads,page", [
    (1 << 27, 1 << 27, 1024), (1 << 30, 1 << 30, 16), (1 << 28, 1 << 30, 64), (2**31 - 1, 2**31 - 1, 1024), (1 << 28, 1, 16), (1, 1 << 28, 16)])
def test_caches_with_too_many_rows(pages, kv_heads, page):
    """The first three products are 2^64, of which 64 bits keep nothing."""
    for name, arguments in (("b200q_cache_write", (empty(3), empty(3), tensor(8192, 1, 3, I32), NONE, None, NONE, NONE, NONE, NONE, 1e-6)),
                            ("b200q_cache_read", (tensor(8192, 1, 3, I32), empty(3), NONE))):
        assert "2^31 - 1 rows" in refused(name, cache(pages, kv_heads, page), *arguments)


@pytest.mark.parametrize("kv_heads,head_dim", [(1 << 26, 64), (1 << 25, 64), (1 << 25, 128), ((1 << 26) + 1, 64), (1 << 24, 128)])
def test_caches_with_too_many_columns(kv_heads, head_dim):
    """Columns of all heads are counted in 32 bits: the first and third of these left 0 of them, and the fourth 64."""
    width = kv_heads * head_dim % 2**32
    width = width if width < 2**31 else 0
    write = (empty(3, width), empty(3, width), tensor(8192, 1, 3, I32), NONE, None, NONE, NONE, NONE, NONE, 1e-6)
    assert "2^31 - 1 columns" in refused("b200q_cache_write", cache(1, kv_heads, 16, head_dim), *write)
    assert "2^31 - 1 columns" in refused("b200q_cache_read", cache(1, kv_heads, 16, head_dim), tensor(8192, 1, 3, I32), empty(3, width), NONE)


def test_outputs_over_the_plan_are_refused():
    """Rows that are written while others still take their angles from there."""
    from tests.test_cache_cpu import cache as small, plan, write
    rotary, positions, at = plan(), tensor(9000, 1, 3, I32), 1 << 29
    x, out = tensor(0, 3, 128), tensor(at - 512, 3, 128)  # rows of 256 bytes: the third begins at the plan
    assert "overlaps its plan" in refused("b200q_rotary", x, positions, rotary, 64, out)
    assert "overlaps its plan" in refused("b200q_rotary", x, positions, rotary, 64, tensor(at + 254, 3, 128))
    assert refused("b200q_rotary", x, positions, rotary, 64, tensor(at + 256, 3, 128)) == ""  # 32 pairs of 8 bytes end there
    assert refused("b200q_rotary", x, positions, rotary, 64, tensor(at - 768, 3, 128)) == ""
    assert "overlaps another operand" in write(rotary=rotary, positions=positions, q=tensor(20000, 3, 128), q_out=out)
    assert "overlaps the cache" in write(small(at=at - 4096), rotary=rotary, positions=positions)


def test_groups_of_too_many_heads_are_refused():
    """Which token a query row belongs to is found by an fp32 product; from 2^23 heads to a cached one on it may name the next."""
    from tests.test_cache_cpu import attention, cache as small
    for heads, refusal in ((1 << 20, ""), ((1 << 20) + 1, "2^20 query heads"), (1 << 24, "2^20 query heads")):
        one = dict(queries=tensor(0, 1, heads * 64), output=tensor(1 << 36, 1, heads * 64), pages=tensor(1 << 37, 1, 5, I32), lengths=tensor(1 << 38, 1, 1, I32))
        got = attention(small(kv_heads=1, at=1 << 39), **one)
        assert got == "" if not refusal else refusal in got


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(16, 8, 1), (32, 1, 1), (8, 1, 4), (64, 2, 1), (16, 8, 16)])
def test_steps_that_a_default_context_is_enough_for(heads, kv_heads, tokens, head_dim):
    """Without a prefix, and with up to 32 query rows to a cached head and sequence."""
    from breeze_tts_cpp_b200 import ops
    for sequences in (1, 64, 10000):
        assert ops.attention_workspace(tokens * sequences, sequences, heads, kv_heads, head_dim) <= 8 << 20


def test_steps_that_ask_for_more():
    from breeze_tts_cpp_b200 import ops
    assert ops.attention_workspace(1, 1, 64, 1, 128) > 8 << 20  # 64 heads to a cached one take partial sums of 64 rows
    assert ops.attention_workspace(64, 64, 16, 8, 128, prefix=True) > 8 << 20
