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


def test_gelu_tails():
    """gelu of values set by the input (z1 = v, z2 = 1): to a relative 1e-3 down to -12,
    where the 24 bits of 1 + erf have long been lost, and one rounding; its slope, by
    way of dx, to 2e-6 and the roundings of dz, of its kept factor and of dx."""
    v = torch.cat([torch.linspace(-12, 12, 1023), torch.tensor([0.0])]).to(BF).to(DEV)
    x = torch.zeros(v.numel(), 64, device=DEV, dtype=BF)
    x[:, 0], x[:, 1] = v, 1.0
    w1, w2 = (torch.zeros(8, 64, device=DEV, dtype=BF) for _ in range(2))
    w1[0, 0] = w2[0, 1] = 1.0
    x.requires_grad_()
    h = gated_linear(x, w1, w2, True)
    dh = torch.zeros_like(h)
    dh[:, 0] = 1.0
    dx, = torch.autograd.grad(h, x, dh)
    z = v.double()
    cdf = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    value = z * cdf
    assert ((h[:, 0].double() - value).abs() <= (U + 1.1e-3) * value.abs()).all()
    assert not h[:, 1:].any()
    slope = cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    assert ((dx[:, 0].double() - slope).abs() <= (2.02 * U + 2.0 ** -16) * slope.abs() + 2e-6).all()


def test_gradient_against_differences():
    """The product is quadratic in x and in each weight linear (identity): along a
    direction exact in bf16, central differences are the gradient but for the outputs'
    roundings, u |h| each."""
    M, I, H = 40, 136, 72
    x, w1, w2, dh = _case(M, I, H, seed=7)
    got = _grads(x, w1, w2, False, dh)
    g = torch.Generator().manual_seed(8)
    for i, n in enumerate(("dx", "dw1", "dw2")):
        ops = [x, w1, w2]
        step = (torch.randint(0, 2, ops[i].shape, generator=g) * 2 - 1).to(DEV) * 2.0 ** -3
        lo, hi = ((ops[i].float() + s * step).to(BF) for s in (-1, 1))
        with torch.no_grad():
            a, b = (gated_linear(*ops[:i], t, *ops[i + 1:], False).double() for t in (lo, hi))
        # the steps as bf16 holds them
        want = ((b - a) * dh.double()).sum()
        moved = (hi.double() - lo.double())
        have = (got[n].double() * moved).sum()
        noise = U * ((a.abs() + b.abs()) * dh.double().abs()).square().sum().sqrt()
        if n == "dx":  # quadratic: the midpoint is not x where the two steps round apart
            noise = noise + ((lo.double() + hi.double()) / 2 - x.double()).abs().max() * 64 * I
        assert abs(have - want) <= 4 * noise + U * (got[n].double() * moved).norm() * 2, n


@pytest.mark.parametrize("gelu", [False, True])
def test_near_the_streamed_product(gelu):
    """gated's values (each step rounded to bf16): within three roundings."""
    x, w1, w2, _ = _case(5, 640, 264, seed=9)
    a, b = gated_linear(x, w1, w2, gelu).double(), gated(x, w1, w2, gelu).double()
    z1, z2 = (x.double() @ w.double().t() for w in (w1, w2))
    assert ((a - b).abs() <= 4 * U * (z1.abs() + 0.2) * z2.abs() + 4 * U * a.abs()).all()


def test_forms_of_call():
    """Leading dimensions, strided and unaligned operands, weights of two strides, an
    expanded upstream gradient, one gradient asked for, no rows: the same values."""
    M, I, H = 24, 136, 72
    x, w1, w2, dh = _case(M, I, H, seed=11)
    want = _grads(x, w1, w2, True, dh)
    wide = torch.zeros(I, H + 16, dtype=BF, device=DEV)
    wide[:, 8:H + 8] = w2
    odd = torch.zeros(M * H + 3, dtype=BF, device=DEV)[3:].view(M, H).copy_(x)
    got = _grads(odd, w1, wide[:, 8:H + 8], True, dh.t().contiguous().t())
    assert all(torch.equal(got[n], want[n]) for n in want)
    lead = gated_linear(x.view(2, 3, 4, H), w1, w2, True)
    assert lead.shape == (2, 3, 4, I) and torch.equal(lead.view(M, I), want["h"])
    xs = x.clone().requires_grad_()
    gated_linear(xs, w1, w2, True).sum().backward()
    ones = _grads(x, w1, w2, True, torch.ones_like(dh))
    assert torch.equal(xs.grad, ones["dx"])
    for i, n in enumerate(("dx", "dw1", "dw2")):
        ops = [x.clone(), w1.clone(), w2.clone()]
        ops[i].requires_grad_()
        gated_linear(*ops, True).backward(dh)
        assert torch.equal(ops[i].grad, want[n]), n
    w = w1.clone().requires_grad_()
    none = gated_linear(x[:0], w, w2, False)
    assert none.shape == (0, I) and not torch.autograd.grad(none.sum(), w)[0].any()
    # the same weight twice: its gradient is both
    both = gated_linear(x, w, w, False)
    got = torch.autograd.grad(both, w, dh)[0]
    twice = _grads(x, w1, w1, False, dh)
    assert ((got.float() - twice["dw1"].float() - twice["dw2"].float()).abs()
            <= 2 * U * got.float().abs() + 1e-30).all()


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("M,I,H", [(777, 2056, 1032), (2048, 1288, 1032)])
def test_same_bits_with_and_without_a_gradient(M, I, H, gelu):
    x, w1, w2, _ = _case(M, I, H, seed=14)
    with torch.no_grad():
        want = gated_linear(x, w1, w2, gelu)
    assert torch.equal(gated_linear(x.requires_grad_(), w1, w2, gelu), want)


def test_nothing_spreads_between_rows():
    """A row of NaN or infinities reaches its own outputs only (and the weights'
    gradients)."""
    x, w1, w2, dh = _case(130, 136, 72, seed=12)
    want = _grads(x, w1, w2, True, dh)
    x[64], x[65, 3] = float("nan"), float("inf")
    got = _grads(x, w1, w2, True, dh)
    rows = torch.ones(130, dtype=torch.bool, device=DEV)
    rows[64:66] = False
    for n in ("h", "dx"):
        assert torch.equal(got[n][rows], want[n][rows]), n
    assert got["h"][64].isnan().all()


def test_repeats_bit_for_bit_in_a_graph():
    """Replays of a captured forward and backward pass, with eager work between, give the
    eager bits; the split sums (few tiles) too."""
    for M, I, H in ((300, 264, 328), (5, 1920, 640)):
        x, w1, w2, dh = _case(M, I, H, seed=13)
        leaves = [t.detach().clone().requires_grad_() for t in (x, w1, w2)]

        def step():
            h = gated_linear(*leaves, True)
            return (h.detach(), *torch.autograd.grad(h, leaves, dh))

        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            with torch.cuda.graph(graph, stream=side):
                outs = step()
        torch.cuda.synchronize()
        for rep in range(3):
            with torch.no_grad():
                leaves[0].copy_(x * (rep + 1))
            graph.replay()
            torch.cuda.synchronize()
            eager = _grads(x * (rep + 1), w1, w2, True, dh)
            assert all(torch.equal(a, b) for a, b in zip(outs, eager.values())), (M, rep)
