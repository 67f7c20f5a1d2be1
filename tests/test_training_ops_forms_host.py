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


UNSUPPORTED = 2


def test_more_workgroups_than_a_launch_takes_are_refused():
    """A launch counts its threads in 32 bits: what takes more is refused before the first of
    a call's launches, by both passes alike."""
    lib, n, at = _lib.lib(), None, 4096  # (an aligned address that is never read)

    def attention(T, nseq, heads, kv, backward):
        if not backward:
            return lib.evo2_packed_attention(at, heads * 64, 64, at, kv * 64, 64, at, kv * 64, 64, at, nseq,
                                             at, n, n, T, heads, kv, 64, 0.1, n)
        return lib.evo2_packed_attention_backward(
            at, heads * 64, 64, at, heads * 64, 64, at, kv * 64, 64, at, kv * 64, 64, at, nseq, at, at, at, at,
            1 << 62, at, at, at, T, heads, kv, 64, 0.1, n)

    for backward in (False, True):
        assert attention(8, (1 << 19) - 1, 32, 32, backward) == UNSUPPORTED
        assert attention(1 << 20, 600000, 32, 8, backward) == UNSUPPORTED
        assert attention(1 << 29, 0, 4, 4, backward) == UNSUPPORTED
    assert b"workgroups" in lib.evo2_last_error()
    rc = lib.evo2_linear_loss(at, 8, at, 8, at, -100, 2, at, at, at, at, at, 1 << 62, 1 << 28, 8, 8, n)
    assert rc == UNSUPPORTED
    # dh's sums over pieces: a thread for eight columns
    rc = lib.evo2_linear_loss_backward(at, 1 << 15, at, 1 << 15, at, -100, at, at, 0, n, at, at, at, 1 << 62,
                                       1 << 20, 9000, 1 << 15, n)
    assert rc == UNSUPPORTED
    # the elementwise gradient: a thread for eight columns
    rc = lib.evo2_gated_linear_backward(at, 1 << 15, at, 8, at, at, 8, at, at, at, at, at, 1 << 62,
                                        1 << 20, 1 << 15, 8, n)
    assert rc == UNSUPPORTED


@pytest.mark.parametrize("shape", [(5, 3), (14,), (15, 1), (3, 1, 5), (3, 4)])
def test_training_targets_of_another_shape_are_refused(shape):
    """Among them those of as many entries, which would be taken in another order."""
    from evo2_flash_amd.model import Evo2DecodeModel

    tokens = torch.zeros(3, 5, dtype=torch.int64)
    with pytest.raises(ValueError, match="tokens' shape"):
        Evo2DecodeModel.training_loss(None, tokens, torch.zeros(shape, dtype=torch.int64))
