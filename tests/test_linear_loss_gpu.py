"""loss.linear_cross_entropy and its gradients against 64-bit arithmetic.

Bounds (u = 2^-8, half a bf16 step; e = 2^-24): a logit is an fp32 sum of H products,
off by dz = (H + 2) e sum |h w|; its exponential relative to the row's log-sum-exp by
that much (twice: z and lse) plus the rounding of the exponent's argument, |z - lse| e.
d is rounded to bf16 once and enters dh and dw with at most u sum |d w|.
"""

import pytest
import torch

from evo2_flash_amd.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U, E = 2.0 ** -8, 2.0 ** -24
IGNORE = -100


def _case(T, V, H, seed, dev=1.3, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g).to(BF).to(DEV)
    w = (torch.randn(V, H, generator=g) * dev / H ** 0.5).to(BF).to(DEV)
    t = torch.randint(V, (T,), generator=g)
    t = torch.where(torch.rand(T, generator=g) < ignored, IGNORE, t).to(DEV)
    return h, w, t, torch.rand(T, generator=g).to(DEV)


def _exact(h, w, t, reduction, grad):
    """{name: (value, bound)} in 64 bits."""
    h, w, t, grad = (x.detach().cpu() for x in (h, w, t, grad))
    h, w, grad = h.double(), w.double(), grad.double()
    T, live = h.shape[0], t != IGNORE
    z, s = h @ w.t(), h.abs() @ w.abs().t()
    lse = torch.logsumexp(z, 1)
    dz = (h.shape[1] + 2) * E * s.amax(1)
    row, idx = torch.arange(T), t.clamp(min=0)
    nll = torch.where(live, lse - z[row, idx], 0.0)
    en = 3 * dz + 16 * E * (lse.abs() + nll.abs() + 1)
    n = live.sum().clamp(min=1)
    weight = torch.where(live, grad if reduction == "none" else torch.ones(T), 0.0)
    if reduction == "mean":
        weight = weight / n
    p = torch.exp(z - lse[:, None])
    onehot = torch.zeros_like(p)
    onehot[row, idx] = 1.0
    d = (p - onehot) * weight[:, None]
    # the exponent's argument z log2 e - lse log2 e, each rounded
    arg = (2 * dz + 4 * E * lse.abs())[:, None] + 4 * E * (z.abs() + (z - lse[:, None]).abs())
    ed = U * d.abs() + weight[:, None] * (p * (2 * arg + 4 * E)) + 4 * E * d.abs()
    loss = {"none": (nll, en), "sum": (nll.sum(), en.sum()),
            "mean": (nll.sum() / n, en.sum() / n + E * nll.sum() / n)}[reduction]
    dh, dw = d @ w, d.t() @ h
    return {"loss": (loss[0], loss[1] + 1e-30),
            "dh": (dh, U * dh.abs() + ed @ w.abs() + 2 * (w.shape[0] + 66) * E * (d.abs() @ w.abs())),
            "dw": (dw, U * dw.abs() + ed.t() @ h.abs() + 2 * (T + 66) * E * (d.abs().t() @ h.abs()))}


def _check(got, want, what):
    for n, t in got.items():
        v, bound = want[n]
        off = (t.detach().cpu().double() - v).abs()
        assert bool((off <= bound * (1 + 2 * U) + 1e-38).all()), (
            what, n, float((off / (bound + 1e-30)).max()))


def _run(h, w, t, reduction, grad):
    h, w = (x.detach().requires_grad_() for x in (h, w))
    loss = linear_cross_entropy(h, w, t, IGNORE, reduction)
    g = grad if reduction == "none" else torch.ones_like(loss)
    return dict(zip(("loss", "dh", "dw"), (loss, *torch.autograd.grad(loss, (h, w), g))))


SIZES = [(1, 2, 8), (1, 512, 64), (3, 7, 72), (32, 130, 128), (65, 512, 200), (300, 512, 264),
         (129, 1000, 520), (700, 4099, 136), (2100, 512, 328), (1, 40000, 64), (17, 20001, 72),
         (600, 33000, 64), (17000, 9000, 16)]


@pytest.mark.parametrize("T,V,H", SIZES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_against_64_bits(T, V, H, reduction):
    if T * V > 1 << 24 and reduction != "mean":
        pytest.skip("the pieces do not depend on the reduction")
    h, w, t, grad = _case(T, V, H, seed=T + V + H)
    t[0] = V - 1
    print(f"linear_cross_entropy {T} {V} {H} {reduction}", flush=True)
    want = _exact(h, w, t, reduction, grad)
    with torch.no_grad():
        _check({"loss": linear_cross_entropy(h, w, t, IGNORE, reduction)}, want, "forward")
    _check(_run(h, w, t, reduction, grad), want, "training")
