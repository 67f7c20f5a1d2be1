"""sample_tokens on long rows of one value beside masked tokens: the cuts and the draw part them
exactly where the settings say (fractions that floating point holds, and even counts)."""

import math

import pytest
import torch

from evo2_flash_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5000, 9000, 20012, 131072, 200004, 1 << 20])
@pytest.mark.parametrize("value", [0.0, 0.3, -7.7, 1.5])
def test_equal_logits(value, V, dtype):
    g = torch.Generator().manual_seed(V)
    u = torch.tensor([0.0, 0.125, 0.5, 0.75, 1 - 2.0 ** -24, 1.0])
    for masked in (0.0, 0.5, 0.99, 0.9999):
        z = torch.full((V,), value)
        z[torch.rand(V, generator=g) < masked] = float("-inf")
        at = (z > float("-inf")).nonzero()[:, 0]
        at = at[:len(at) // 8 * 8]  # (so that eighths and halves of them are whole numbers)
        if not len(at):
            continue
        z = torch.full((V,), float("-inf")).index_fill(0, at, value).to(dtype)
        for B in (6, 3):
            for t in (1.0, 0.8, 3.3):
                for s in ({}, {"top_p": 0.5}, {"top_p": 0.25, "min_p": 0.5}, {"min_p": 1.0}, {"top_k": len(at) // 2},
                          {"top_k": len(at) // 2, "top_p": 0.5}):
                    n = len(at)
                    n = min(n, s.get("top_k", n))
                    n = math.ceil(s.get("top_p", 1.0) * n) if n else n
                    got = sample_tokens(z.to(DEV)[None].expand(B, V), u[-B:].to(DEV), temperature=t, **s).tolist()
                    want = [int(at[min(math.floor(x * n), n - 1)]) for x in u[-B:].tolist()]
                    assert got == want, (masked, t, s, n)
