"""The gated product's weight gradients where the rows they walk lie past 2^31 elements and
2^32 bytes: those of the last rows, which alone have an upstream gradient, against the same
rows on their own (fp32 sums in another order; each rounded once, u = 2^-8)."""

import pytest
import torch

from evo2_flash_amd.linear import gated_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U = 2.0 ** -8


@pytest.mark.parametrize("gelu", [False, True])
def test_gated_linear_weights(gelu):
    M, I, H, tail = 70000, 32768, 64, 300
    g = torch.Generator(device=DEV).manual_seed(4)
    x, w1, w2 = (torch.randn(n, H, generator=g, device=DEV).to(BF) for n in (M, I, I))
    assert (M - tail) * 2 * I > 1 << 31
    print(f"gated_linear, weights' gradients {M} x {I}", flush=True)
    dh = torch.zeros(M, I, dtype=BF, device=DEV)
    dh[-tail:] = (torch.randn(tail, I, generator=g, device=DEV) * 0.01).to(BF)
    got = []
    for rows in (slice(None), slice(M - tail, None)):
        leaves = [t.clone().requires_grad_() for t in (x[rows], w1, w2)]
        got.append(torch.autograd.grad(gated_linear(*leaves, gelu), leaves[1:], dh[rows]))
    for a, b in zip(*got):
        a, b = a.double(), b.double()
        assert b.norm() > 0 and (a - b).norm() <= 2 * U * b.norm()
