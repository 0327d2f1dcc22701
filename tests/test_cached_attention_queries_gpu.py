"""How exactly the attention over the quantized cache takes its queries: rows with one element far above the others, in a column where the keys are zero."""
import pytest
import torch

from breeze_tts_cpp_b200 import ops
from tests.cache_reference import check, held
from tests.test_cached_attention_gpu import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [9, 13])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", [ops.I8, ops.FP8])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("counts", [[1, 1], [70, 40]])  # both kernels
def test_elements_far_below_their_rows_largest(ctx_factory, counts, head_dim, fmt, dtype, power):
    """BF16 elements are taken to within 2^-25 of the power of two of their row's largest, which is nothing where they are within 2^-17 of it; F16 ones
    are taken as they are. A score is off by at most that times the sum of the key's magnitudes, and a weight by as much twice over."""
    batch = Batch(50, [n + 100 for n in counts], counts, heads=4, kv_heads=2, head_dim=head_dim, page=16, fmt=fmt, dtype=dtype)
    column = 5
    batch.cache.keys[..., column] = 0
    batch.q.view(-1, 4, head_dim)[..., column] = 2.0**power
    want, bound = batch.want()
    if dtype == torch.bfloat16 and power > 9:
        numbers = torch.isfinite(batch.cache.key_scales.cpu())  # what no length reaches is not
        magnitudes = (held(batch.cache.keys.cpu(), fmt).abs().sum(-1) * batch.cache.key_scales.cpu().double())[numbers]
        values = (held(batch.cache.values.cpu(), fmt).abs().amax(-1) * batch.cache.value_scales.cpu().double())[numbers]
        delta = 2.0 ** (power - 25) * magnitudes.max() * head_dim**-0.5
        bound = bound + (want.abs() + values.max()) * torch.expm1(2 * delta)
    check(batch.run(ctx_factory("int8")), want, bound)
