"""Operands whose rows the ABI's (rows, columns, stride) cannot say, without a GPU: fake tensors, whose addresses nobody gets to ask for."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from breeze_tts_cpp_b200 import ops


@pytest.mark.parametrize("shape", [(3, 128), (2, 1), (1000, 4)])
def test_expanded_rows_are_refused(shape):
    """A stride of 0 says dense rows: what the call would touch lies behind the one row that there is."""
    with FakeTensorMode():
        one = torch.empty(1, shape[1], dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match="overlap"):
            ops._tensor(one.expand(shape))
        with pytest.raises(ValueError, match="overlap"):
            ops._tensor(one[0].expand(shape))


def test_windows_are_refused():
    with FakeTensorMode():
        with pytest.raises(ValueError, match="overlap"):
            ops._tensor(torch.empty(64, dtype=torch.int32, device="cuda").unfold(0, 16, 4))


@pytest.mark.parametrize("shape,columns", [((2, 2**32 + 128), 128), ((3, 2**31), 16), ((2**32 + 3, 16), 16), ((1, 2**32 + 16), 2**32 + 16)])
def test_sizes_past_32_bits_are_refused(shape, columns):
    """Their low 32 bits may be sizes that the call takes."""
    with FakeTensorMode():
        with pytest.raises(ValueError, match="2\\^31"):
            ops._tensor(torch.empty(shape, dtype=torch.bfloat16, device="cuda")[:, :columns])
