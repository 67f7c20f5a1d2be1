"""What the training operators' wrappers hand to the kernels, and what the C entries refuse
before a launch, without a GPU."""

import pytest
import torch

from evo2_flash_amd import _lib

BF = torch.bfloat16


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("stride", [8, 16, (1 << 22) - 8, 1 << 22, (1 << 22) + 8])
def test_rows_as_the_matrix_kernels_take_them(rows, stride):
    """Rows 2^22 elements apart or further are copied, single ones too; nearer ones stay."""
    base = torch.arange(stride + 64, dtype=torch.float32).to(BF)
    t = base[:stride + 8].as_strided((rows, 8), (stride, 1))
    got = _lib.rows16(t)
    assert torch.equal(got, t) and got.stride(1) == 1 and got.stride(0) < 1 << 22
    assert (got.data_ptr() == t.data_ptr()) == (stride < 1 << 22)
