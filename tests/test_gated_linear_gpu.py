"""linear.gated_linear and its gradients against 64-bit arithmetic.

Bounds (u = 2^-8, half a bf16 step; e = 2^-24): a bf16 result is off by u |v|, an fp32
sum of K products by (K + 2) e sum |a b|.  The products z1 and z2 are kept in fp32, so
d1 and d2 differ from the exact ones by one rounding u (and the fp32 errors); entering
dx and dw they give at most u sum |d w|.
"""

import pytest
import torch

from evo2_flash_amd.linear import gated, gated_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U, E = 2.0 ** -8, 2.0 ** -24


def _case(M, I, H, seed, dev=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, H, generator=g).to(BF).to(DEV)
    w1, w2 = ((torch.randn(I, H, generator=g) * dev / H ** 0.5).to(BF).to(DEV) for _ in range(2))
    return x, w1, w2, torch.randn(M, I, generator=g).to(BF).to(DEV)


def _exact(x, w1, w2, gelu, dh):
    """{name: (value, bound)} in 64 bits."""
    x, w1, w2, dh = (t.detach().cpu().double() for t in (x, w1, w2, dh))
    z1, z2 = x @ w1.t(), x @ w2.t()
    s1, s2 = x.abs() @ w1.abs().t(), x.abs() @ w2.abs().t()
    k = (x.shape[1] + 2) * E
    if gelu:
        cdf = 0.5 * (1 + torch.erf(z1 / 2 ** 0.5))
        a, slope = z1 * cdf, cdf + z1 * torch.exp(-z1 * z1 / 2) / (2 * torch.pi) ** 0.5
    else:
        a, slope = z1, torch.ones_like(z1)
    # |gelu'| <= 1.13 and |gelu''| <= 0.8; the fp32 erf and exp add a few e
    da, dslope = 1.13 * k * s1 + 8 * E * z1.abs(), gelu * (0.8 * k * s1 + 16 * E)
    h = a * z2
    eh = U * h.abs() + da * z2.abs() + 2 * k * s2 * a.abs() + 4 * E * h.abs()
    d1, d2 = dh * z2 * slope, dh * a
    e1 = U * d1.abs() + dh.abs() * (k * s2 * slope.abs() + z2.abs() * dslope) * 1.01 + 4 * E * d1.abs()
    e2 = U * d2.abs() + dh.abs() * da * 1.01 + 4 * E * d2.abs()
    dx, sx = d1 @ w1 + d2 @ w2, d1.abs() @ w1.abs() + d2.abs() @ w2.abs()
    ex = U * dx.abs() + e1 @ w1.abs() + e2 @ w2.abs() + 2 * (2 * w1.shape[0] + 66) * E * sx
    out = {"h": (h, eh), "dx": (dx, ex)}
    for n, d, e in (("dw1", d1, e1), ("dw2", d2, e2)):
        out[n] = (d.t() @ x, U * (d.t() @ x).abs() + e.t() @ x.abs()
                  + 2 * (x.shape[0] + 66) * E * (d.abs().t() @ x.abs()))
    return out


def _check(got, want, what):
    for n, t in got.items():
        v, bound = want[n]
        off = (t.detach().cpu().double() - v).abs()
        assert bool((off <= bound * (1 + 2 * U) + 1e-38).all()), (
            what, n, float((off / (bound + 1e-30)).max()))


def _grads(x, w1, w2, gelu, dh):
    leaves = [t.detach().requires_grad_() for t in (x, w1, w2)]
    h = gated_linear(*leaves, gelu)
    return dict(zip(("h", "dx", "dw1", "dw2"), (h, *torch.autograd.grad(h, leaves, dh))))


SIZES = [(1, 8, 8), (1, 128, 64), (2, 136, 72), (5, 1920, 640), (63, 264, 328), (64, 128, 128),
         (65, 120, 2056), (129, 640, 200), (200, 1288, 968), (257, 520, 264), (700, 328, 1032),
         (1500, 904, 520)]


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("M,I,H", SIZES)
def test_against_64_bits(M, I, H, gelu):
    x, w1, w2, dh = _case(M, I, H, seed=M + I + H)
    print(f"gated_linear {M} {I} {H} {gelu}", flush=True)
    want = _exact(x, w1, w2, gelu, dh)
    with torch.no_grad():
        _check({"h": gated_linear(x, w1, w2, gelu)}, want, "forward")
    _check(_grads(x, w1, w2, gelu, dh), want, "training")
