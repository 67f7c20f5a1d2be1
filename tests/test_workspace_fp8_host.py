"""workspace_fp8: one workspace for calls of fewer sequences and fewer tokens as well."""

import pytest

from evo2_flash_amd import _lib
from evo2_flash_amd.kv_fp8 import workspace_fp8


@pytest.mark.parametrize("B,heads,kv,hd,cols,n,shared", [
    (16, 32, 4, 64, 545, 8, 0), (16, 32, 8, 128, 545, 8, 0), (5, 32, 32, 128, 251, 4, 128), (3, 4, 4, 64, 1, 3, 0),
    (16, 32, 4, 64, 545, 1, 0),
])
def test_smaller_calls_fit(B, heads, kv, hd, cols, n, shared):
    need = _lib.lib().evo2_decode_attention_fp8_workspace_bytes
    have = workspace_fp8(B, heads, kv, hd, cols, "cpu", n=n, shared_pages=shared).numel()
    most = max(need(b, m, heads, kv, hd, cols, s) for b in range(1, B + 1) for m in range(1, n + 1) for s in (0, shared))
    assert have == max(most, 16)
