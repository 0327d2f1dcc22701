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


@pytest.mark.parametrize("counts", [None, [40, 33, 7]])
def test_prefix_behind_its_producers_without_a_pause(counts):
    """The second pass of a call starts before the first is over, yet behind everything that the call reads: queries, keys and lengths that the launch in
    front of it has just written, in the same buffers step after step."""
    lengths = [200, 150, 90]
    batch = Batch(41, lengths, counts, heads=8, kv_heads=4, head_dim=128, page=64, prefix=600)
    rows, steps = batch.q.shape[0], 60
    g = torch.Generator().manual_seed(2)
    queries = torch.randn(steps, *batch.q.shape, generator=g).bfloat16().cuda()
    keys = torch.randn(steps, rows, 4 * 128, generator=g).bfloat16().cuda()
    # Every step's rows go to the first slots of the prefix, which all queries read, and of the sequences.
    places = torch.cat((batch.prefix_pages[:9].long()[:, None] * 64 + torch.arange(64), batch.pages[:, :1].long() * 64 + torch.arange(64))).flatten()
    slots = torch.stack([places[torch.randperm(len(places), generator=g)[:rows]] for _ in range(steps)]).to(torch.int32).cuda()
    positions, rotary = torch.arange(rows, dtype=torch.int32, device="cuda"), ops.Rotary.plan(128)
    stored = [getattr(batch.cache, n).clone() for n in ("keys", "values", "key_scales", "value_scales")]
    context = ops.Context("int8", workspace_bytes=64 << 20)
    q, out, pages = torch.empty_like(queries[0]), batch.out.cuda(), batch.pages.cuda()
    of = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    offsets = None if counts is None else torch.tensor(batch.offsets, dtype=torch.int32, device="cuda")
    prefix_pages, prefix_length = batch.prefix_pages.cuda(), batch.prefix_length.cuda()

    def run(pause):
        for n, x in zip(("keys", "values", "key_scales", "value_scales"), stored):
            getattr(batch.cache, n).copy_(x)
        outs = torch.zeros(steps, *out.shape, dtype=out.dtype, device="cuda")
        torch.cuda.synchronize()
        for i in range(steps):
            context.cache_write(batch.cache, keys[i], keys[i], slots[i], positions, rotary, queries[i], q)
            if pause:
                torch.cuda.synchronize()
            context.cached_attention(q, batch.cache, pages, of, outs[i], query_offsets=offsets, prefix_pages=prefix_pages, prefix_length=prefix_length)
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert context.status() == 0
        return outs

    want = run(True)
    assert torch.isfinite(want).all() and not torch.equal(want[0], want[1])
    for _ in range(5):
        assert torch.equal(run(False), want)
    context.close()


@pytest.mark.parametrize("counts", [[1] * 9 + [70] + [1] * 3, [1, 200, 0, 1, 90, 1], [300] + [1] * 30])
@pytest.mark.parametrize("prefix", [None, 90])
def test_decode_rows_beside_chunks_of_prompts(ctx_factory, counts, prefix):
    """One call for both; the batch's average says which kernel takes it: the first and third the one for few rows, the second the other."""
    g = torch.Generator().manual_seed(len(counts))
    lengths = [n + int(torch.randint(0, 200, (1,), generator=g)) for n in counts]
    batch = Batch(42, lengths, counts, heads=4, kv_heads=2, head_dim=64, page=16, prefix=prefix, spare_rows=2)
    check(batch.run(ctx_factory("int8")), *batch.want())
