"""The training operators where element offsets pass 2^31 and byte offsets 2^32: the
last rows against the same rows on their own.  (A row's sums may be taken in another
order there: fp32 sums, then one rounding to bf16, u = 2^-8; what enters a second
product as bf16 adds u of its absolute sum, here below twice the values' norm.)"""

import pytest
import torch

from evo2_flash_amd.attention import packed_attention
from evo2_flash_amd.linear import gated_linear
from evo2_flash_amd.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U = 2.0 ** -8


def _near(a, b):
    a, b = a.double(), b.double()
    return (a - b).norm() <= 2 * U * b.norm()


def test_gated_linear():
    M, I, H, tail = 70000, 32768, 64, 300
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w1, w2 = (torch.randn(n, H, generator=g, device=DEV).to(BF) for n in (M, I, I))
    print(f"gated_linear {M} x {I}", flush=True)
    assert M * I > 1 << 31
    xs = x.clone().requires_grad_()
    h = gated_linear(xs, w1, w2, True)
    dh = torch.zeros_like(h)
    dh[-tail:] = torch.randn(tail, I, generator=g, device=DEV).to(BF) * 0.01
    dx = torch.autograd.grad(h, xs, dh)[0]
    last = x[-tail:].clone().requires_grad_()
    want = gated_linear(last, w1, w2, True)
    assert _near(h[-tail:], want)
    assert _near(dx[-tail:], torch.autograd.grad(want, last, dh[-tail:])[0])
    assert not dx[:-tail].any()


def test_linear_cross_entropy():
    T, V, H, tail = 300000, 8192, 64, 257
    g = torch.Generator(device=DEV).manual_seed(2)
    h = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w = (torch.randn(V, H, generator=g, device=DEV) * 0.2).to(BF)
    t = torch.randint(V, (T,), generator=g, device=DEV)
    print(f"linear_cross_entropy {T} x {V}", flush=True)
    assert T * V > 1 << 31
    grad = torch.zeros(T, device=DEV)
    grad[-tail:] = torch.rand(tail, generator=g, device=DEV)
    got = []
    for rows in (slice(None), slice(T - tail, None)):
        hs, ws = h[rows].clone().requires_grad_(), w.clone().requires_grad_()
        nll = linear_cross_entropy(hs, ws, t[rows], reduction="none")
        got.append((nll[-tail:].detach(), *torch.autograd.grad(nll, (hs, ws), grad[rows])))
    (nll, dh, dw), (nll1, dh1, dw1) = got
    assert (nll - nll1).abs().max() <= 1e-4
    assert _near(dh[-tail:], dh1) and _near(dw, dw1) and not dh[:-tail].any()


def test_packed_attention():
    """Rows 65536 elements apart: the last sequences lie past 4 GB."""
    T, heads, hd, step = 40000, 2, 128, 1 << 16
    g = torch.Generator(device=DEV).manual_seed(3)
    rows = torch.empty(T, step, dtype=BF, device=DEV)
    tail = torch.randn(3, 200, heads, hd, generator=g, device=DEV).to(BF)
    q, k, v = (rows[:, 8 + 512 * i:8 + 512 * i + heads * hd].view(T, heads, hd) for i in range(3))
    for t, s in zip((q, k, v), tail):
        t[-200:] = s
    assert q.stride(0) == step and (T - 200) * step * 2 > 1 << 32
    # (the rows before hold no sequence)
    cu = torch.tensor([T - 200, T - 200, T - 70, T], dtype=torch.int32, device=DEV)
    d = torch.zeros(T, heads, hd, dtype=BF, device=DEV)
    d[-200:] = torch.randn(200, heads, hd, generator=g, device=DEV).to(BF)
    print(f"packed_attention rows {step} apart", flush=True)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, cu, 0.1)
    grads = torch.autograd.grad(out, leaves, d)
    small = [t.clone().requires_grad_() for t in tail]
    want = packed_attention(*small, torch.tensor([0, 130, 200], device=DEV), 0.1)
    assert torch.equal(out[-200:], want) and not out[:-200].any()
    for a, b in zip(grads, torch.autograd.grad(want, small, d[-200:])):
        assert torch.equal(a[-200:], b) and not a[:-200].any()
