"""Attention over the quantized cache against its 64-bit form, element by element within a derived bound."""
import pytest
import torch

from breeze_tts_cpp_b200 import _lib, ops
from tests.cache_reference import attention, check

pytestmark = pytest.mark.gpu
FORMATS = {"int8": ops.I8, "fp8": ops.FP8}
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


class Batch:
    """A cache, its tables and queries. Whatever no length reaches is garbage: NaN scales, bytes that are no numbers, pages that do not exist."""

    def __init__(self, seed, lengths, counts=None, heads=4, kv_heads=2, head_dim=128, page=16, fmt=ops.I8, dtype=torch.bfloat16, prefix=None,
                 spare_rows=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        needed = [-(-max(n, 0) // page) for n in lengths]
        shared = -(-prefix // page) if prefix is not None else 0
        pages = sum(needed) + shared + 1
        shape = (pages, kv_heads, page, head_dim)
        bytes_ = [torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2)]
        if fmt == ops.FP8:
            for x in bytes_:
                x[(x & 0x7f) == 0x7f] = 0x7e
        scales = [torch.exp(torch.randn(shape[:3], generator=g) * spread) * (0.02 if fmt == ops.I8 else 0.005) for _ in range(2)]
        order = torch.randperm(pages, generator=g).to(torch.int32)
        columns = max(max(needed), 1) + 1
        self.pages = torch.full((len(lengths), columns), 10**6, dtype=torch.int32)
        used = torch.zeros(pages, page, dtype=torch.bool)
        at = 0
        tables = []
        for b, count in enumerate(needed):
            self.pages[b, :count] = order[at: at + count]
            tables.append((order[at: at + count], max(lengths[b], 0)))
            at += count
        self.prefix_pages = self.prefix_length = None
        if prefix is not None:
            self.prefix_pages = torch.full((shared + 1,), -7, dtype=torch.int32)
            self.prefix_pages[:shared] = order[at: at + shared]
            self.prefix_length = torch.tensor([prefix], dtype=torch.int32)
            tables.append((order[at: at + shared], prefix))
        for table, length in tables:
            for i, p in enumerate(table.tolist()):
                used[p, : max(0, min(page, length - i * page))] = True
        for x in bytes_:
            x.transpose(1, 2)[~used] = 0x7f
        for x in scales:
            x.transpose(1, 2)[~used] = float("nan")
        self.cache = ops.CacheView(*(x.cuda() for x in bytes_), *(x.cuda() for x in scales), fmt)
        self.lengths, self.prefix = lengths, prefix or 0
        rows = len(lengths) if counts is None else sum(counts)
        self.offsets = None if counts is None else [sum(counts[:i]) for i in range(len(counts) + 1)]
        self.q = (torch.randn(rows + spare_rows, heads * head_dim, generator=g) * 2).to(dtype)
        self.out = torch.full_like(self.q, 5.0)

    def run(self, ctx, out=None, q=None, **more):
        out = self.out.cuda() if out is None else out
        ctx.cached_attention(self.q.cuda() if q is None else q, self.cache, self.pages.cuda(),
                             torch.tensor(self.lengths, dtype=torch.int32, device="cuda"), out,
                             query_offsets=None if self.offsets is None else torch.tensor(self.offsets, dtype=torch.int32, device="cuda"),
                             prefix_pages=None if self.prefix_pages is None else self.prefix_pages.cuda(),
                             prefix_length=None if self.prefix_length is None else self.prefix_length.cuda(), **more)
        torch.cuda.synchronize()
        assert ctx.status() == 0
        return out

    def want(self, scale=None):
        return attention(self.q, self.cache, self.pages, self.lengths, self.out, scale, self.offsets, self.prefix_pages, self.prefix)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,heads,kv_heads,head_dim,page", [
    ([1], 1, 1, 64, 16), ([16], 2, 1, 128, 16), ([17, 0, 128, 1], 4, 2, 128, 16), ([129, 127, 300], 8, 1, 64, 32),
    ([2000], 16, 8, 128, 64), ([10, 300, 20, 30, 129, 500, 7, 90] * 6, 8, 4, 64, 16), ([5, 640, 0, 33, 257, 1], 12, 3, 128, 256), ([700, 90], 16, 1, 64, 1024), ([400] * 9, 10, 2, 128, 128)])
def test_one_query_per_sequence(ctx_factory, lengths, heads, kv_heads, head_dim, page, fmt, dtype):
    batch = Batch(len(lengths), lengths, None, heads, kv_heads, head_dim, page, FORMATS[fmt], DTYPES[dtype])
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,head_dim,page", [
    ([40], [40], 2, 1, 128, 16), ([300, 7, 0, 130], [5, 7, 0, 1], 4, 2, 128, 32), ([260, 129], [130, 65], 3, 1, 64, 64),
    ([3, 500], [9, 2], 8, 4, 64, 16), ([1100], [3], 16, 8, 128, 128),
    # More segments than multiprocessors, many of a single tile between longer ones.
    ([100, 700, 90], [60, 50, 60], 16, 8, 64, 32), ([130, 60, 257, 40], [40, 33, 70, 40], 8, 8, 128, 16)])
def test_some_queries_per_sequence(ctx_factory, lengths, counts, heads, kv_heads, head_dim, page, fmt, dtype):
    # The fourth has more query rows than cached tokens: the first ones see nothing. Rows behind the last sequence stay.
    batch = Batch(sum(counts), lengths, counts, heads, kv_heads, head_dim, page, FORMATS[fmt], DTYPES[dtype], spare_rows=3)
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,counts,prefix,heads,kv_heads,head_dim,page", [
    ([1, 30, 200], None, 77, 4, 2, 128, 16), ([0, 0], None, 513, 2, 1, 64, 32), ([9, 140], None, 0, 2, 2, 128, 64),
    ([9, 140, 6], [2, 5, 0], 300, 4, 1, 64, 16), ([20] * 70, None, 1025, 4, 2, 128, 128), ([1], None, 1, 1, 1, 128, 1024)])
def test_shared_prefix(ctx_factory, lengths, counts, prefix, heads, kv_heads, head_dim, page, fmt, dtype):
    batch = Batch(prefix, lengths, counts, heads, kv_heads, head_dim, page, FORMATS[fmt], DTYPES[dtype], prefix=prefix,
                  spare_rows=2 if counts else 0)
    check(batch.run(ctx_factory("int8")), *batch.want())


def test_many_sequences(ctx_factory):
    """More than a warp adds up by itself."""
    g = torch.Generator().manual_seed(1)
    batch = Batch(20, torch.randint(0, 300, (700,), generator=g).tolist(), None, heads=2, kv_heads=2, head_dim=64, page=32)
    check(batch.run(ctx_factory("int8")), *batch.want())
    batch = Batch(21, torch.randint(0, 40, (300,), generator=g).tolist(), torch.randint(0, 3, (300,), generator=g).tolist(), heads=2, kv_heads=1,
                  head_dim=64, page=16, prefix=50, spare_rows=1)
    check(batch.run(ctx_factory("int8")), *batch.want())


def test_parts_that_only_one_team_has_tiles_of(ctx_factory):
    """Over a thousand short segments of 128 query rows between longer ones, many to a multiprocessor and call after call without a pause."""
    g = torch.Generator().manual_seed(5)
    counts = torch.randint(20, 200, (40,), generator=g).tolist()
    batch = Batch(23, [n + (1500 if b % 7 == 3 else 0) for b, n in enumerate(counts)], counts, heads=32, kv_heads=16, head_dim=64, page=64)
    first = batch.run(ctx_factory("int8"))
    out = batch.out.cuda()
    q, pages, lengths = batch.q.cuda(), batch.pages.cuda(), torch.tensor(batch.lengths, dtype=torch.int32, device="cuda")
    offsets = torch.tensor(batch.offsets, dtype=torch.int32, device="cuda")
    ctx = ctx_factory("int8")
    for _ in range(200):
        ctx.cached_attention(q, batch.cache, pages, lengths, out, query_offsets=offsets)
    torch.cuda.synchronize()
    assert ctx.status() == 0 and torch.equal(out, first)
    some = [0, 7, 20]  # sequences, in 64 bits
    for b in some:
        rows = slice(batch.offsets[b], batch.offsets[b + 1])
        want, bound = attention(batch.q[rows, :256], ops.CacheView(batch.cache.keys[:, :2].contiguous(), batch.cache.values[:, :2].contiguous(),
                                batch.cache.key_scales[:, :2].contiguous(), batch.cache.value_scales[:, :2].contiguous(), ops.I8),
                                batch.pages[b: b + 1], batch.lengths[b: b + 1], batch.out[rows, :256], None, [0, counts[b]])
        check(first[rows, :256], want, bound)


@pytest.mark.parametrize("prefix", [None, 20])
def test_no_queries_at_all(ctx_factory, prefix):
    batch = Batch(22, [30, 0], [0, 0], spare_rows=2, prefix=prefix)
    assert (batch.run(ctx_factory("int8")) == 5).all()


def test_lengths_beyond_the_tables_are_clamped(ctx_factory):
    batch = Batch(3, [48, 32], None, page=16)
    batch.pages = batch.pages[:, :2].contiguous()  # 32 positions each
    batch.lengths = [48, -5]
    check(batch.run(ctx_factory("int8")), *batch.want())


def test_positions_on_missing_pages_read_as_nan(ctx_factory):
    batch = Batch(4, [100, 100], [2, 2], page=16)
    batch.pages[0, 6] = 10**6  # positions 96 to 99: both queries of the first sequence see some of them
    batch.pages[1, 1] = -1
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_row_that_is_not_a_number_reaches_only_those_who_see_it(ctx_factory, fmt):
    batch = Batch(5, [64, 64], [4, 4], fmt=FORMATS[fmt], page=16)
    page = batch.pages[0, 3].item()
    batch.cache.value_scales[page, 1, 14] = float("nan")  # position 62 of the first sequence: seen by its last two queries
    batch.cache.key_scales[batch.pages[1, 3].item(), 0, 15] = float("nan")  # position 63 of the second: by the last
    got, (want, bound) = batch.run(ctx_factory("int8")), batch.want()
    # The 64-bit form of the masked rows never reads them, the operator's must not either.
    check(got, want, bound)
    assert torch.isnan(want).any() and not torch.isnan(want).all()


@pytest.mark.parametrize("spread", [8.0, 20.0])
def test_scales_far_apart(ctx_factory, spread):
    """Value scales over 1e-20 to 1e20: the weights' range must not depend on them."""
    batch = Batch(6, [300, 40], None, fmt=ops.I8, dtype=torch.bfloat16, page=16)
    g = torch.Generator().manual_seed(9)
    batch.cache.value_scales.mul_(torch.exp(torch.randn(batch.cache.value_scales.shape, generator=g) * spread / 2).cuda())
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("power", [-90, 100])
def test_queries_of_any_magnitude(ctx_factory, power):
    batch = Batch(7, [200, 60], None, dtype=torch.bfloat16, page=16)
    batch.q = (batch.q.double() * 2.0**power).bfloat16()
    scale = 2.0**-power * 0.05
    check(batch.run(ctx_factory("int8"), scale=scale), *batch.want(scale))


def test_strided_rows_and_scale(ctx_factory):
    batch = Batch(8, [130, 31, 77], None, heads=4, kv_heads=2, head_dim=64, page=32)
    want, bound = batch.want(0.3)
    for shift in (0, 3):  # an odd start has no 16-byte alignment
        packed = torch.full((3, 4 * 64 + 40), 9.0, dtype=torch.bfloat16, device="cuda")
        held = torch.full((3, 4 * 64 + 24), 9.0, dtype=torch.bfloat16, device="cuda")
        q, out = packed[:, shift: shift + 256], held[:, shift: shift + 256]
        q.copy_(batch.q)
        check(batch.run(ctx_factory("int8"), out=out, q=q, scale=0.3), want, bound)
        assert (held[:, :shift] == 9).all() and (held[:, shift + 256:] == 9).all()


def test_same_outcome_every_time(ctx_factory):
    batch = Batch(10, [1500, 3, 800], [3, 1, 8], heads=8, kv_heads=2, prefix=900)
    first = batch.run(ctx_factory("int8"))
    for _ in range(3):
        assert torch.equal(batch.run(ctx_factory("int8")), first)


def test_refusals(ctx_factory):
    ctx, batch = ctx_factory("int8"), Batch(11, [20, 20], None)
    q, pages, lengths = batch.q.cuda(), batch.pages.cuda(), torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    for call, text in ((lambda: ctx.cached_attention(q, batch.cache, pages, lengths, q), "overlaps"),
                       (lambda: ctx.cached_attention(q, batch.cache, pages, lengths, out.half()), "type mismatch"),
                       (lambda: ctx.cached_attention(q, batch.cache, pages, lengths[:1], out), "one per sequence"),
                       (lambda: ctx.cached_attention(q[:1], batch.cache, pages, lengths, out[:1]), "one query row"),
                       (lambda: ctx.cached_attention(q, batch.cache, pages, lengths, out, prefix_pages=pages[0]), "prefix needs"),
                       (lambda: ctx.cached_attention(q, batch.cache, pages, lengths, out, scale=float("nan")), "not finite")):
        with pytest.raises(_lib.B200QError, match=text):
            call()
    small = ops.Context("int8", workspace_bytes=64 << 10)
    with pytest.raises(_lib.B200QError, match="workspace of"):
        small.cached_attention(q, batch.cache, pages, lengths, out)
    small.close()


def many(counts=(70, 40), **other):
    """More than 32 query rows of a cached head: the tensor memory's kernel."""
    lengths = [n + 100 for n in counts]
    return Batch(30, lengths, list(counts), **{"heads": 4, "kv_heads": 2, "page": 16, **other})


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_rows_with_missing_pages_and_rows_that_are_no_numbers(ctx_factory, fmt, head_dim):
    batch = many(fmt=FORMATS[fmt], head_dim=head_dim)
    batch.pages[0, 6] = 10**6  # positions 96 to 111 of 170: seen by all
    batch.pages[1, 8] = -3  # positions 128 to 139: by the last twelve queries
    page = batch.pages[1, 7].item()
    batch.cache.value_scales[page, 1, 10] = float("nan")  # position 122: by the last eighteen, of one cached head
    batch.cache.key_scales[page, 0, 11] = float("nan")
    got, (want, bound) = batch.run(ctx_factory("int8")), batch.want()
    check(got, want, bound)
    assert torch.isnan(want[:70]).all() and not torch.isnan(want[70:90]).any() and torch.isnan(want[-1]).all()


@pytest.mark.parametrize("spread", [8.0, 20.0])
def test_many_rows_with_scales_far_apart(ctx_factory, spread):
    batch = many(fmt=ops.I8)
    g = torch.Generator().manual_seed(9)
    batch.cache.value_scales.mul_(torch.exp(torch.randn(batch.cache.value_scales.shape, generator=g) * spread / 2).cuda())
    check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("power", [-90, 100])
def test_many_rows_of_any_magnitude(ctx_factory, power):
    batch = many()
    batch.q = (batch.q.double() * 2.0**power).bfloat16()
    scale = 2.0**-power * 0.05
    check(batch.run(ctx_factory("int8"), scale=scale), *batch.want(scale))


def test_many_rows_beside_a_row_that_is_huge_or_infinite(ctx_factory):
    """BF16 rows enter fp16 each by a power of two of its own: a row 2^28 above the others, or one with an infinity, costs those nothing. (Nothing is
    asked of these rows: scores of 2^30 are known to within 2^6 in fp32, so exp of them to within a factor of 2^64.)"""
    batch = many()
    batch.q = batch.q.clone()
    batch.q[5] = (batch.q[5].double() * 2.0**28).bfloat16()
    batch.q[9, 3] = float("inf")
    batch.q[81, 70] = float("-inf")
    batch.q[90] = (batch.q[90].double() * 2.0**28).bfloat16()
    got, (want, bound) = batch.run(ctx_factory("int8")), batch.want()
    others = [r for r in range(110) if r not in (5, 9, 81, 90)]
    check(got[others], want[others], bound[others])


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_strided(ctx_factory, dtype):
    batch = many(head_dim=64, dtype=DTYPES[dtype])
    want, bound = batch.want(0.3)
    rows = batch.q.shape[0]
    for shift in (0, 3, 8):  # 16-byte alignment for the last, 32 for the first only
        packed = torch.full((rows, 4 * 64 + 40), 9.0, dtype=batch.q.dtype, device="cuda")
        held = torch.full((rows, 4 * 64 + 24), 9.0, dtype=batch.q.dtype, device="cuda")
        q, out = packed[:, shift: shift + 256], held[:, shift: shift + 256]
        q.copy_(batch.q)
        check(batch.run(ctx_factory("int8"), out=out, q=q, scale=0.3), want, bound)
        assert (held[:, :shift] == 9).all() and (held[:, shift + 256:] == 9).all()


def test_references_that_rise_late(ctx_factory):
    """Scores that grow by far more than the weights' range from tile to tile: the outputs so far are rescaled, again and again."""
    for batch in (many((130,), page=64, head_dim=128), Batch(31, [700], None, heads=2, kv_heads=1, page=64, head_dim=128),
                  many((40, 30), page=64, head_dim=64, prefix=600)):
        shape = batch.cache.key_scales.shape
        tables = [t for t in ([batch.pages] if batch.prefix_pages is None else [batch.prefix_pages[None], batch.pages])]
        for table in tables:
            for row in table.tolist():
                for i, p in enumerate(row):
                    if 0 <= p < shape[0]:
                        batch.cache.key_scales[p] *= 1.6 ** i
        check(batch.run(ctx_factory("int8")), *batch.want())


@pytest.mark.parametrize("prefix", [None, 900])
@pytest.mark.parametrize("counts", [None, [40, 33, 1]])
def test_values_whose_scale_is_zero(ctx_factory, counts, prefix):
    """A cache filled by its owner may hold zero scales, runs of tiles of them: they weigh in the sum, wherever the shares end."""
    batch = Batch(34, [1500, 900, 300], counts, heads=2, kv_heads=1, page=64, prefix=prefix)
    for b, runs in ((0, [(0, 12)]), (1, [(0, 15)]), (2, [(1, 3)])):
        for first, last in runs:
            batch.cache.value_scales[batch.pages[b, first:last].clamp(max=batch.cache.value_scales.shape[0] - 1).long()] = 0.0
    if prefix:
        batch.cache.value_scales[batch.prefix_pages[3:9].long()] = 0.0
    context = ops.Context("int8", workspace_bytes=64 << 20)
    check(batch.run(context), *batch.want())
    context.close()


def test_strided_page_tables(ctx_factory):
    batch = Batch(32, [130, 31, 77, 0], None, page=32)
    wide = torch.full((4, 3 * batch.pages.shape[1] + 1), 7 * 10**5, dtype=torch.int32)
    part = wide[:, 2: 2 + batch.pages.shape[1]]
    part.copy_(batch.pages)
    on_device = wide.cuda()[:, 2: 2 + batch.pages.shape[1]]
    out = batch.out.cuda()
    ctx = ctx_factory("int8")
    ctx.cached_attention(batch.q.cuda(), batch.cache, on_device, torch.tensor(batch.lengths, dtype=torch.int32, device="cuda"), out)
    check(out, *batch.want())


def test_offsets_that_are_none(ctx_factory):
    """Offsets that fall, or lie outside of the rows, name rows inside of them or none: nothing else is written, nothing waits for good."""
    batch = Batch(33, [60, 60, 60], [2, 2, 2], spare_rows=4)
    lengths = torch.tensor(batch.lengths, dtype=torch.int32, device="cuda")
    ctx, held = ctx_factory("int8"), torch.full((14, batch.q.shape[1]), 5.0, dtype=batch.q.dtype, device="cuda")
    for offsets in ([0, 4, 2, 6], [0, 2, 4, 99], [-3, 2, 4, 6], [6, 4, 2, 0], [2**31 - 1, -(2**31), 5, 5]):
        ctx.cached_attention(batch.q.cuda(), batch.cache, batch.pages.cuda(), lengths, held[2:12],
                             query_offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert ctx.status() == 0 and (held[:2] == 5).all() and (held[12:] == 5).all()
