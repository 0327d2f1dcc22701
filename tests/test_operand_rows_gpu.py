"""Operands whose rows the ABI cannot say, through every way into the library: refused before anything is launched."""
import pytest
import torch

from breeze_tts_cpp_b200 import ops

pytestmark = pytest.mark.gpu


def test_expanded_rows_are_refused(ctx_factory):
    ctx = ctx_factory("int8")
    cache = ops.CacheView.empty(4, 2, 16, 64, ops.I8)
    cache.keys.fill_(1), cache.values.fill_(1), cache.key_scales.fill_(1), cache.value_scales.fill_(1)
    x, index = torch.randn(3, 128, device="cuda").bfloat16(), torch.zeros(3, dtype=torch.int32, device="cuda")
    out, rotary = torch.empty_like(x), ops.Rotary.plan(64)
    row, page = x[:1].expand(3, -1), torch.arange(2, dtype=torch.int32, device="cuda")[None].expand(3, -1)
    lengths = torch.full((3,), 20, dtype=torch.int32, device="cuda")
    for call in (lambda: ctx.rotary(row, index, rotary, 64), lambda: ctx.rotary(x, index, rotary, 64, out=row),
                 lambda: ctx.cache_write(cache, row, x, index), lambda: ctx.cache_write(cache, x, row, index),
                 lambda: ctx.cache_write(cache, x, x, index, q=row, q_out=out), lambda: ctx.cache_read(cache, index, row, None),
                 lambda: ctx.cached_attention(row, cache, page.contiguous(), lengths, out),
                 lambda: ctx.cached_attention(x, cache, page, lengths, out),
                 lambda: ctx.quantize_rows(row, ops.RowScaledView.empty(3, 128, ops.I8)),
                 lambda: ops.Linear(ctx, [x[:1].expand(64, -1)], max_rows=3)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # One row may have any stride, and copies of the refused ones are taken.
    assert torch.equal(ctx.rotary(x[:1].expand(1, -1), index[:1], rotary, 64), ctx.rotary(row.contiguous(), index, rotary, 64)[:1])
    ctx.cached_attention(x, cache, page.contiguous(), lengths, out)
    assert torch.isfinite(out).all()
