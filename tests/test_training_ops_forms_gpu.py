"""Forms of call of the training operators beside those of their own tests."""

import pytest
import torch

from evo2_flash_amd.linear import gated_linear
from evo2_flash_amd.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("B", [1, 3])
def test_the_last_position_of_long_sequences(B):
    """Rows that lie 2^22 elements apart and further: the values of the same rows on their
    own, the weights' and the gradients' views among them."""
    L, H, I = 8200, 512, 72
    assert L * H >= 1 << 22
    g = torch.Generator(device=DEV).manual_seed(B)
    x = torch.randn(B, L, H, generator=g, device=DEV).to(BF)
    w = (torch.randn(2, I, H, generator=g, device=DEV) * 0.05).to(BF)
    t = torch.randint(I, (B,), generator=g, device=DEV)
    far = torch.empty(B, 1 << 22, dtype=BF, device=DEV)[:, :I]
    far.copy_(torch.randn(B, I, generator=g, device=DEV))
    for rows in (x[:, -1], x[:, -1:].squeeze(1)):
        got = []
        for r, d in ((rows, far), (rows.contiguous().clone(), far.clone())):
            leaves = [v.detach().requires_grad_() for v in (r, *w)]
            h = gated_linear(*leaves, True)
            got.append([h, *torch.autograd.grad(h, leaves, d)])
            loss = linear_cross_entropy(*leaves[:2], t, reduction="none")
            got[-1] += [loss, *torch.autograd.grad(loss, leaves[:2], torch.ones_like(loss))]
        assert all(torch.equal(a, b) for a, b in zip(*got))
    tall = torch.empty(8, 1 << 22, dtype=BF, device=DEV)[:, :H].copy_(w[0, :8])
    assert torch.equal(gated_linear(x[:, -1], tall, tall, False),
                       gated_linear(x[:, -1], w[0, :8], w[0, :8], False))
