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


def test_gradient_against_differences():
    """Central differences of the fp32 loss over steps exact in bf16: off by the third
    derivative's s^2 / 6 (|w|^3 <= (4 / 9)^3 per entry: below 1e-3 here) and the loss's own
    error over the step."""
    T, V, H = 5, 300, 72
    h, w, t, _ = _case(T, V, H, seed=1, ignored=0.0)
    h, w = (x.mul(8).round().div(8).to(BF) for x in (h, w.mul(4)))  # exact under the steps
    got = _run(h, w, t, "sum", None)
    s = 2.0 ** -4
    for name, x in (("dh", h), ("dw", w)):
        for r, c in ((0, 0), (4, 71), (t[2].item() if name == "dw" else 2, 9)):
            loss = []
            for step in (s, -s):
                moved = x.clone()
                moved[r, c] += step
                assert float(moved[r, c] - x[r, c]) == step
                args = (moved, w) if name == "dh" else (h, moved)
                with torch.no_grad():
                    loss.append(linear_cross_entropy(*args, t, IGNORE, "sum").item())
            want = (loss[0] - loss[1]) / (2 * s)
            g = got[name][r, c].item()
            third = x.abs().max().item() ** 3 if name == "dh" else h.abs().max().item() ** 3 * T
            third = min(third, 64.0)
            assert abs(g - want) <= 4 * U * (1 + abs(g)) + s * s / 6 * third + 2e-5 / s, (name, r, c)


def test_bad_targets_and_ignored_rows():
    """A target outside the vocabulary: NaN in its row's loss and gradient, nowhere else;
    ignored rows: loss 0, no gradient, whatever they hold; no counted row: a NaN mean."""
    for T, V in ((6, 40), (300, 600)):
        h, w, t, grad = _case(T, V, 64, seed=2, ignored=0.0)
        t[1], t[2], t[3] = V, -5, IGNORE
        h[3] = float("inf")
        got = _run(h, w, t, "none", grad)
        bad = torch.tensor([1, 2], device=DEV)
        assert got["loss"][bad].isnan().all() and got["dh"][bad].isnan().all()
        good = torch.ones(T, dtype=torch.bool, device=DEV)
        good[bad] = False
        assert got["loss"][good].isfinite().all() and got["dh"][good].isfinite().all()
        assert got["loss"][3] == 0 and not got["dh"][3].any()
        t[:] = IGNORE
        h[3] = 0
        got = _run(h, w, t, "mean", grad)
        assert got["loss"].isnan() and not got["dh"].any() and not got["dw"].any()


def test_forms_of_call():
    """Leading dimensions, strided and unaligned operands, int32 targets, one gradient
    asked for, an expanded upstream gradient, no rows: the same values."""
    T, V, H = 24, 130, 72
    h, w, t, _ = _case(T, V, H, seed=3)
    want = _run(h, w, t, "mean", None)
    wide = torch.zeros(T, H + 8, dtype=BF, device=DEV)
    wide[:, :H] = h
    odd = torch.zeros(V * H + 1, dtype=BF, device=DEV)[1:].view(V, H).copy_(w)
    got = _run(wide[:, :H], odd, t.to(torch.int32), "mean", None)
    assert all(torch.equal(got[n], want[n]) for n in want)
    lead = linear_cross_entropy(h.view(2, 3, 4, H), w, t.view(2, 3, 4), IGNORE, "none")
    assert lead.shape == (2, 3, 4)
    assert torch.equal(lead.view(-1), linear_cross_entropy(h, w, t, IGNORE, "none"))
    hg = h.clone().requires_grad_()
    linear_cross_entropy(hg, w, t, IGNORE, "none").sum().backward()
    assert (hg.grad.float() - want["dh"].float() * (t != IGNORE).sum()).norm() <= \
        2 * U * hg.grad.float().norm()
    wg = w.clone().requires_grad_()
    linear_cross_entropy(h, wg, t, IGNORE).backward()
    assert torch.equal(wg.grad, want["dw"])
    none = linear_cross_entropy(h[:0], wg, t[:0], IGNORE, "sum")
    assert none.item() == 0 and not torch.autograd.grad(none, wg)[0].any()
    assert linear_cross_entropy(h[:0], w, t[:0], IGNORE).isnan()
    assert linear_cross_entropy(h[:0], w, t[:0], IGNORE, "none").shape == (0,)


def test_repeats_bit_for_bit_in_a_graph_and_on_a_stream():
    """Two calls give the same bits, eagerly, on another stream and replayed from a
    graph with other work between (no atomics)."""
    h, w, t, _ = _case(700, 1000, 264, seed=4)
    want = _run(h, w, t, "mean", None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(h, w, t, "mean", None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    hs, ws = (x.detach().clone().requires_grad_() for x in (h, w))

    def step():
        loss = linear_cross_entropy(hs, ws, t, IGNORE)
        return (loss.detach(), *torch.autograd.grad(loss, (hs, ws)))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    for rep in range(3):
        with torch.no_grad():
            hs.copy_(h * (rep + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(h * (rep + 1), w, t, "mean", None)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager.values())), rep
