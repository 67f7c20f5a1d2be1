"""New and cleared 8-bit caches: zeros with the scale that zeros have, so that a first write
behind a page's start (a decode step on a cleared cache) gets a scale of its own values."""

import pytest
import torch

from evo2_flash_amd.kv_fp8 import Fp8KVCache, read_kv_fp8, rotary_decode_fp8, write_kv_fp8

from _kv_fp8 import exponent

DEV = "cuda"
BF = torch.bfloat16


def _caches(device):
    new, used = Fp8KVCache(3, 2, 64, device), Fp8KVCache(3, 2, 64, device)
    for t in used.tensors[:2]:
        t.view(torch.uint8).fill_(0x55)
    for t in used.tensors[2:]:
        t.fill_(2.0 ** 9)
    used.clear()
    return new, used


def test_scales_of_zeros():
    for cache in _caches("cpu"):
        for codes in cache.tensors[:2]:
            assert not codes.view(torch.uint8).any()
        for scale in cache.tensors[2:]:
            assert scale.dtype == torch.float32 and (scale == 2.0 ** int(exponent(torch.zeros(1, dtype=torch.float64)))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 2.0 ** -12, 2.0 ** -60])
def test_a_first_write_behind_a_pages_start(size):
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[1], [2]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([5, 15], device=DEV)
    rows = (torch.randn(2, 3 * 128, generator=g) * size).to(BF).to(DEV)
    q, k, v = rows.view(2, 1, 3, 2, 64).unbind(2)
    inv = torch.zeros(32, device=DEV)  # no rotation
    for rotary in (False, True):
        for cache in _caches(DEV):
            if rotary:
                rotary_decode_fp8(rows, cache, table, pos, inv, 1.0)
            else:
                write_kv_fp8(k, v, *cache.tensors, table, pos)
            got = read_kv_fp8(*cache.tensors, table, pos + 1, 16)
            for x, y, scale in zip(got, (k, v), cache.tensors[2:]):
                for b, p in enumerate(pos.tolist()):
                    want = y[b, 0].double().cpu()
                    e = exponent(want.abs().amax(1))
                    assert torch.equal(scale[b + 1].double().cpu(), torch.exp2(e))
                    assert not x[b, :p].any() and not x[b, p + 1:].any()
                    # half a step: 2^-4 of the value, or of the subnormal step 2^-9
                    off = (x[b, p].double().cpu() - want).abs()
                    assert (off <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * torch.exp2(e)[:, None]).all()
