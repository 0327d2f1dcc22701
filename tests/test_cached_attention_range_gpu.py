"""The cache operators far out: contexts of 16000 tokens, and a cache whose far end lies past 2^32 bytes and 2^24 rows."""
import pytest
import torch

from breeze_tts_cpp_b200 import ops
from tests.cache_reference import check
from tests.test_cached_attention_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [ops.I8, ops.FP8])
@pytest.mark.parametrize("lengths,counts,prefix,page", [
    ([16001, 5, 12345], None, None, 16), ([16001, 3000], [3, 1], None, 64), ([16001], [40], None, 128), ([300, 16385], [50, 20], None, 32),
    ([20, 3], None, 16001, 64), ([40, 60], [20, 17], 16385, 16)])
def test_long_contexts(lengths, counts, prefix, page, fmt):
    batch = Batch(60, lengths, counts, heads=4, kv_heads=2, head_dim=64, page=page, fmt=fmt, prefix=prefix)
    context = ops.Context("int8", workspace_bytes=64 << 20)
    check(batch.run(context), *batch.want())
    context.close()


FAR = dict(pages=1 << 19, kv_heads=2, page=64, head_dim=128)  # 2^26 rows of 128 bytes


@pytest.fixture(scope="module")
def far_cache():
    # Nothing may read what nobody wrote, and nobody writes anything but the last pages: scales beside them are no numbers.
    shape = (FAR["pages"], FAR["kv_heads"], FAR["page"])
    values = [torch.empty(*shape, FAR["head_dim"], dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full(shape, float("nan"), device="cuda") for _ in range(2)]
    yield ops.CacheView(*values, *scales, ops.I8)
    del values, scales
    torch.cuda.empty_cache()


@pytest.mark.parametrize("counts,prefix", [(None, None), ([50, 30, 40], None), (None, 200), ([50, 30, 40], 70)])
def test_attention_at_the_far_end_of_a_large_cache(far_cache, counts, prefix):
    batch = Batch(61, [300, 77, 150], counts, heads=4, kv_heads=FAR["kv_heads"], head_dim=FAR["head_dim"], page=FAR["page"], prefix=prefix)
    want = batch.want()
    near, first = batch.cache, FAR["pages"] - batch.cache.keys.shape[0]
    for name in ("keys", "values", "key_scales", "value_scales"):
        getattr(far_cache, name)[first:] = getattr(near, name)
    moved = lambda t: None if t is None else torch.where((t >= 0) & (t < near.keys.shape[0]), t + first, t)  # noqa: E731
    batch.cache, batch.pages, batch.prefix_pages = far_cache, moved(batch.pages), moved(batch.prefix_pages)
    context = ops.Context("int8", workspace_bytes=64 << 20)
    check(batch.run(context), *want)
    context.close()


def test_writing_and_reading_at_the_far_end_of_a_large_cache(ctx_factory, far_cache):
    ctx, rows, width = ctx_factory("int8"), 40, FAR["kv_heads"] * FAR["head_dim"]
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(rows, width, generator=g).bfloat16().cuda() for _ in range(2))
    total = FAR["pages"] * FAR["page"]
    slots = (total - 1 - torch.randperm(200, generator=g)[:rows]).to(torch.int32).cuda()
    small = ops.CacheView.empty(1, FAR["kv_heads"], 64, FAR["head_dim"], ops.I8)
    places = torch.arange(rows, dtype=torch.int32, device="cuda")
    read = [torch.empty_like(k) for _ in range(4)]
    for cache, at, out in ((far_cache, slots, read[:2]), (small, places, read[2:])):
        ctx.cache_write(cache, k, v, at)
        ctx.cache_read(cache, at, *out)
    torch.cuda.synchronize()
    assert torch.equal(read[0], read[2]) and torch.equal(read[1], read[3]) and not torch.equal(read[0], read[1])
