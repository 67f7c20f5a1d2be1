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


def _kept(x, w1, w2, gelu):
    """Both factors that the gated product keeps for its gradients, from their planes: the
    high 16 bits of each, then the next eight of both."""
    from evo2_flash_amd.linear import _gated_forward

    planes = _gated_forward(x, w1, w2, gelu, True)[1].to(torch.int32) & 0xffff
    a, b, low = planes
    return [t.view(torch.float32).double()
            for t in ((a << 16) | ((low & 0xff) << 8), (b << 16) | (low & 0xff00))]


@pytest.mark.parametrize("lower", [False, True])
@pytest.mark.parametrize("M", [300, 2048])
def test_kept_factors_are_rounded_to_nearest(M, lower):
    """Products of 24 significant bits, exact in fp32 (a + b 2^-8 + c 2^-16 of 8-bit a, b,
    c): kept to 16 bits, the nearest.  The last eight bits are 128 + an odd number, which
    rounds up, or with `lower` (2^-16 taken off) the odd number, which rounds down; no ties.
    Infinities and NaN stay what they are."""
    g = torch.Generator().manual_seed(M)
    x = torch.zeros(M, 64)
    a, b, c = (torch.randint(0, n, (M,), generator=g) for n in (110, 128, 64))
    x[:, 0], x[:, 1], x[:, 2] = 1 + a / 128, 1 + b / 128, 1 + (2 * c + 1) / 128
    x[:, 3] = float(lower)
    w = torch.zeros(2, 136, 64)
    w[0, :, :4] = torch.tensor([1.0, 2.0 ** -8, 2.0 ** -16, -2.0 ** -16])
    w[1] = -2 * w[0]
    want = x.double() @ w.double().transpose(1, 2)  # z1, z2
    x, w = x.to(BF).to(DEV), w.to(BF).to(DEV)
    print(f"kept factors, {M} rows", flush=True)
    a2, b1 = _kept(x, *w, False)
    for got, z in ((a2, want[1]), (b1, want[0])):
        step = 2.0 ** (torch.floor(torch.log2(z.abs())) - 15)
        assert torch.equal(got.cpu(), torch.round(z / step) * step)
    x[5], x[6, 0] = float("nan"), float("inf")
    for gelu in (False, True):
        a2, b1 = _kept(x, *w, gelu)
        assert a2[5].isnan().all() and b1[5].isnan().all()
        assert (b1[6] == float("inf")).all()
        rest = torch.ones(M, dtype=torch.bool, device=DEV)
        rest[5:7] = False
        assert a2[rest].isfinite().all() and b1[rest].isfinite().all()


@pytest.mark.parametrize("T,V,H", [(17000, 9000, 16), (65600, 8300, 8)])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_loss_over_several_pieces_of_the_vocabulary(T, V, H, reduction):
    """Rows weighted by their own upstream gradient ("none") and by one (the mean is among
    the operator's other sizes), in two pieces, targets in both."""
    g = torch.Generator(device=DEV).manual_seed(T + V)
    h = torch.randn(T, H, generator=g, device=DEV).to(BF)
    w = (torch.randn(V, H, generator=g, device=DEV) * 0.3).to(BF)
    t = torch.randint(V, (T,), generator=g, device=DEV)
    t[::5] = -100
    t[1], t[2] = 0, V - 1
    up = torch.rand(T, generator=g, device=DEV) if reduction == "none" else torch.tensor(0.75, device=DEV)
    print(f"linear_cross_entropy {T} {V} {H} {reduction}", flush=True)
    hs, ws = (v.clone().requires_grad_() for v in (h, w))
    loss = linear_cross_entropy(hs, ws, t, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (hs, ws), up)
    live = t != -100
    weight = torch.where(live, up, 0.0).double()
    want_h, want_w = torch.zeros(T, H, dtype=torch.float64, device=DEV), torch.zeros(V, H, dtype=torch.float64, device=DEV)
    size_h, size_w = torch.zeros_like(want_h), torch.zeros_like(want_w)
    nll = torch.zeros(T, dtype=torch.float64, device=DEV)
    for r0 in range(0, T, 8192):
        r = slice(r0, min(T, r0 + 8192))
        row = torch.arange(r.stop - r.start, device=DEV)
        z = h[r].double() @ w.double().t()
        lse = torch.logsumexp(z, 1)
        nll[r] = torch.where(live[r], lse - z[row, t[r].clamp(min=0)], 0.0)
        d = torch.exp(z - lse[:, None])
        d[row, t[r].clamp(min=0)] -= 1.0
        d *= weight[r, None]
        want_h[r], size_h[r] = d @ w.double(), d.abs() @ w.double().abs()
        want_w += d.t().contiguous() @ h[r].double()
        size_w += d.abs().t().contiguous() @ h[r].double().abs()
    # fp32 logits, |z| and lse below 32: exponents off by 64 e = 2^-18; d to bf16, u of the
    # absolute sums, and a result to bf16, u of itself; fp32 sums of n terms n e of them
    e, u = 2.0 ** -24, 2.0 ** -8
    got = loss.double() if reduction == "none" else loss.double() - nll.sum()
    off = (got - nll).abs().max() if reduction == "none" else got.abs()
    assert off <= 64 * e * (1 if reduction == "none" else T) + e * nll.sum()
    for got, want, size, n in ((dh, want_h, size_h, V), (dw, want_w, size_w, T)):
        bound = u * want.abs() + (u + 2.0 ** -17 + n * e) * size
        assert bool(((got.double() - want).abs() <= bound * (1 + 2 * u) + 1e-38).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_where_infinities_and_nan_reach(hd):
    """Rows the mask parts from a NaN, and that share no tile with it, keep their bits."""
    from evo2_flash_amd.attention import packed_attention

    T, heads, kv = 300, 4, 2
    g = torch.Generator(device=DEV).manual_seed(hd)
    q, k, v, d = (torch.randn(T, n, hd, generator=g, device=DEV).to(BF) for n in (heads, kv, kv, heads))
    cu = torch.tensor([0, 20, 300], dtype=torch.int32, device=DEV)

    def run(*ops):
        leaves = [t.detach().requires_grad_() for t in ops[:3]]
        out = packed_attention(*leaves, cu, 0.1)
        return (out, *torch.autograd.grad(out, leaves, ops[3]))

    want = run(q, k, v, d)
    row = 20 + 150  # in its sequence's 64-row tile from 128, 32-row tile from 128 to 159
    for i in range(4):
        ops = [t.clone() for t in (q, k, v, d)]
        ops[i][row, 0] = float("nan")
        got = run(*ops)
        if i in (1, 2):  # keys and values: queries before the tile
            for n in (0, 1):
                assert torch.equal(got[n][:20 + 128], want[n][:20 + 128]), (i, n)
                assert got[n][row].isnan().any()
        else:  # queries and upstream gradients: keys behind the tile
            for n in (2, 3):
                assert torch.equal(got[n][20 + 160:], want[n][20 + 160:]), (i, n)
                assert torch.equal(got[n][:20], want[n][:20]), (i, n)
                assert got[n][row].isnan().any() or (i, n) == (3, 2)
