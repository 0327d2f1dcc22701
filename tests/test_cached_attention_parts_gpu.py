"""Cached attention as a server calls it: many parts to a multiprocessor, call after call without a pause, decode rows beside prompts, graphs in turn,
pages that are shared, offsets that are none."""
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
    """The few-rows kernel's merge buffers change hands all the time, while one of its two merging warps has less to do than the other, or nothing."""
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


def test_two_graphs_of_one_context_in_turn():
    """Both use the context's workspace, one behind the other: a prefix's two passes, chunks, and eager steps between their replays."""
    side = torch.cuda.Stream()
    context = ops.Context("int8", stream=side, workspace_bytes=64 << 20)
    batches = [Batch(43, [90, 400, 33], None, heads=8, kv_heads=4, prefix=500), Batch(44, [150, 80], [60, 80], heads=4, kv_heads=2),
               Batch(45, [700, 2, 90, 129], None, heads=4, kv_heads=4, head_dim=64)]
    calls, want = [], []
    for batch in batches:
        q, pages, out = batch.q.cuda(), batch.pages.cuda(), batch.out.cuda()
        lengths = torch.tensor(batch.lengths, dtype=torch.int32, device="cuda")
        more = {} if batch.offsets is None else {"query_offsets": torch.tensor(batch.offsets, dtype=torch.int32, device="cuda")}
        if batch.prefix_pages is not None:
            more.update(prefix_pages=batch.prefix_pages.cuda(), prefix_length=batch.prefix_length.cuda())
        calls.append((out, lambda a=(q, batch.cache, pages, lengths, out), more=more: context.cached_attention(*a, **more)))
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(side):
        for (out, call), batch in zip(calls, batches):
            call()
            side.synchronize()
            check(out, *batch.want())
            want.append(out.clone())
        for _, call in calls[:2]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                call()
        for out, _ in calls:
            out.fill_(5.0)
        for _ in range(100):
            graphs[0].replay()
            graphs[1].replay()
            calls[2][1]()
            graphs[0].replay()
            calls[1][1]()
    torch.cuda.synchronize()
    assert context.status() == 0 and all(torch.equal(out, w) for (out, _), w in zip(calls, want))
    graphs.clear()
    context.close()


def test_many_sequences_of_many_rows(ctx_factory):
    """More sequences than a warp adds up by itself, for the kernel of many rows."""
    g = torch.Generator().manual_seed(6)
    counts = torch.randint(0, 45, (300,), generator=g).tolist()
    batch = Batch(46, [n + b % 90 for b, n in enumerate(counts)], counts, heads=2, kv_heads=1, head_dim=64, page=16, spare_rows=1)
    assert sum(counts) * 2 > 32 * len(counts)
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("counts", [None, [40, 20, 33]])
def test_pages_that_several_sequences_name(ctx_factory, counts):
    """The same page in several tables, twice in one, and in the prefix."""
    batch = Batch(47, [100, 80, 64], counts, heads=4, kv_heads=2, head_dim=64, page=16, prefix=64)
    batch.pages[1, :5] = batch.pages[0, :5]
    batch.pages[2, :4] = batch.pages[0, 2]
    batch.prefix_pages[1] = batch.pages[0, 3]
    batch.prefix_pages[3] = batch.pages[0, 3]
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("counts,prefix", [([60, 50, 40], None), ([60, 50, 40], 100), ([2, 2, 2], 100)])
def test_offsets_that_are_none(ctx_factory, counts, prefix):
    """Whatever offsets name, nothing outside of the rows is written and nothing waits for good; calls with right ones are right again."""
    batch = Batch(48, [n + 60 for n in counts], counts, heads=4, kv_heads=2, head_dim=64, page=16, prefix=prefix, spare_rows=4)
    ctx, rows = ctx_factory("int8"), batch.q.shape[0]
    lengths, held = torch.tensor(batch.lengths, dtype=torch.int32, device="cuda"), torch.full((rows + 4, 256), 5.0, dtype=batch.q.dtype, device="cuda")
    more = {} if prefix is None else {"prefix_pages": batch.prefix_pages.cuda(), "prefix_length": batch.prefix_length.cuda()}
    half = rows // 2
    for offsets in ([0, rows, 2, half], [0, 2, half, 10**6], [-3, 2, half, rows], [rows, half, 2, 0], [2**31 - 1, -(2**31), 5, 5], [half, half + 1, rows, rows]):
        ctx.cached_attention(batch.q.cuda(), batch.cache, batch.pages.cuda(), lengths, held[2: 2 + rows],
                             query_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), **more)
        torch.cuda.synchronize()
        assert ctx.status() == 0 and (held[:2] == 5).all() and (held[2 + rows:] == 5).all()
    check(batch.run(ctx), *batch.want())
