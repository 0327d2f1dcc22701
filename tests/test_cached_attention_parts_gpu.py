"""The few-rows attention with many parts to a multiprocessor, call after call without a pause: its merge buffers change hands all the time, while
one of the two merging warps has less to do than the other, or nothing."""
import pytest
import torch

from breeze_tts_cpp_b200 import ops
from tests.cache_reference import attention, check
from tests.test_cached_attention_gpu import Batch

pytestmark = pytest.mark.gpu


def some_of(batch, first, sequences):
    """What some sequences' rows have to be, in 64 bits, from a cache that holds their pages only."""
    tables = batch.pages[sequences]
    if batch.prefix_pages is not None:
        tables = torch.cat((tables.flatten(), batch.prefix_pages))
    kept = torch.unique(tables[(tables >= 0) & (tables < batch.cache.keys.shape[0])].long())
    place = torch.full((10**6 + 1,), 10**6, dtype=torch.int32)
    place[kept] = torch.arange(len(kept), dtype=torch.int32)
    parts = (getattr(batch.cache, n)[kept.cuda()] for n in ("keys", "values", "key_scales", "value_scales"))
    prefix = place[batch.prefix_pages.clamp(min=0).long()] if batch.prefix_pages is not None else None
    want, bound = attention(batch.q[sequences], ops.CacheView(*parts, batch.cache.format), place[batch.pages[sequences].long()],
                            [batch.lengths[b] for b in sequences], batch.out[sequences], None, None, prefix, batch.prefix)
    check(first[sequences], want, bound)


@pytest.mark.parametrize("heads,kv_heads,head_dim,prefix", [
    (8, 8, 64, None), (16, 8, 64, None), (8, 8, 128, None), (16, 8, 128, None), (24, 8, 64, None), (24, 8, 128, None), (32, 8, 64, None),
    (32, 8, 128, None), (8, 8, 64, 70), (16, 8, 64, 300), (16, 8, 128, 70)])
def test_many_parts_without_a_pause(heads, kv_heads, head_dim, prefix):
    g = torch.Generator().manual_seed(heads + head_dim)
    lengths = torch.randint(1, 300, (1100,), generator=g).tolist()
    batch = Batch(40, lengths, None, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=64, prefix=prefix)
    context = ops.Context("int8", workspace_bytes=256 << 20)
    first = batch.run(context)
    some_of(batch, first, [0, 5, 147, 148, 777, 1099])
    q, pages, lengths = batch.q.cuda(), batch.pages.cuda(), torch.tensor(batch.lengths, dtype=torch.int32, device="cuda")
    more = {} if prefix is None else {"prefix_pages": batch.prefix_pages.cuda(), "prefix_length": batch.prefix_length.cuda()}
    outs = torch.full((50, *first.shape), 5.0, dtype=first.dtype, device="cuda")
    for _ in range(6):
        outs.fill_(5.0)
        torch.cuda.synchronize()
        for out in outs:
            context.cached_attention(q, batch.cache, pages, lengths, out, **more)
        torch.cuda.synchronize()
        assert context.status() == 0 and all(torch.equal(out, first) for out in outs)
    context.close()
