"""sample_tokens on long rows whose parts lie tens of nats apart, so that the slices a row is
taken in have largest logits of very different weight: a draw that falls into a far part takes
a token of that part, and numbers of 1 and above the last token kept.

The reference holds weights and running sums in 80-bit floating point.  The kernel's sums:

* a token's weight is off by at most half a step of its slice's units, 2^-62 of the largest
  times V rounded up to a power of two: 8192 of them by V 2^-49 of the slice's largest, all by
  V 2^-49 of the total.  Where a cut goes through its values the units are the row's, of 2^-49
  of the largest or 2^-61 of the sum: V 2^-50 of the total for all;
* a slice's sum loses at most a step of the row's units, and each of its 256 bins where a cut is
  looked for: 256 V / 4096 of them;
* so a running sum is off by less than E = V 2^-48 of the total.

A number u draws a token whose part of the running sum u times the total reaches within 3 E
(its own sum, the total and top-p's border); top-p keeps tokens whose front is below p times
the total within E."""

import numpy as np
import pytest
import torch

from evo2_flash_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAST = 1.0 - 2.0 ** -24
US = [0.0, 0.5, 1.0 - 2.0 ** -20, LAST, 1.0, 3.0]


def _rows(z, n):
    return z.to(DEV)[None].expand(n, -1)


def _check(z, us=US, t=1.0, k=0, p=1.0, m=0.0):
    """The tokens drawn, all rows in one call; checked, and a few rows' in another one (slices
    are of 8192 or 4096 logits by the number of rows)."""
    V, E = len(z), len(z) * 2.0 ** -48
    got = [sample_tokens(_rows(z, len(u)), torch.tensor(u, device=DEV), t, k, p, m).tolist()
           for u in (us, us[-3:])]
    f = lambda x: np.longdouble(float(torch.tensor(x, dtype=torch.float32)))  # noqa: E731
    x = z.double().numpy()
    w = np.exp((x.astype(np.longdouble) - x.max()) / f(t))
    order = np.argsort(-x, kind="stable")
    order = order[np.isfinite(x[order])]
    if k:
        order = order[:k]
    allowed = np.zeros(V, bool)
    if p < 1:
        run = np.cumsum(w[order])
        before = run - w[order]
        allowed[order[before <= (f(p) + E) * run[-1]]] = True
        order = order[:max(int((before < f(p) * run[-1]).sum()), 1)]
    else:
        allowed[order] = True
    allowed &= w >= min(f(m), 1)
    order = order[w[order] >= min(f(m), 1)]
    kept = np.zeros(V, np.longdouble)
    kept[order] = w[order]
    run = np.cumsum(kept)
    total = run[-1]
    # of two steps of the kernel's at least (a step of the sum: 2^-61 of a bound on it, which
    # with top-k is up to eight times the sum)
    counted = order[w[order] >= max(2.0 ** -48, total * 2.0 ** -57)].max()
    for u, token in (*zip(us, got[0]), *zip(us[-3:], got[1])):
        assert allowed[token], (u, token)
        at = min(f(u), 1) * total
        assert run[token] - kept[token] <= at + 3 * E * total, (u, token)
        assert run[token] >= at - 3 * E * total, (u, token)
        if u >= 1 and p >= 1:
            assert token >= counted, (u, token, counted)
    return got[0]


def _peaked(V, depth, at, dtype):
    z = torch.full((V,), -depth)
    z[at] = 0.0
    return z.to(dtype)


SETTINGS = [{}, {"m": 1e-15}, {"p": LAST}, {"k": -1}, {"p": 0.9999999, "m": 1e-15}, {"t": 1.5}]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [131072, 1 << 20])
@pytest.mark.parametrize("depth", [20.0, 30.1, 33.9, 50.0])
@pytest.mark.parametrize("at", [0, -1])
def test_a_peak_over_a_flat_tail(at, depth, V, dtype):
    z = _peaked(V, depth, at, dtype)
    for s in SETTINGS:
        s = dict(s)
        if "k" in s:
            s["k"] = V - 7
        _check(z, **s)


def test_the_number_next_to_one_draws_from_the_tail():
    """A tail of 2^20 - 1 tokens of e^-30.1 weighs 2^-23.4: two thirds of it lie behind
    1 - 2^-24 of the total.  Those in the peak's slice, of up to 8192 (0.8% of the row), count
    for nothing; one in the row's units is 47 steps of 2^-49, within half a step of its weight,
    1.1% of those two thirds."""
    V = 1 << 20
    z = _peaked(V, 30.1, 0, torch.float32)
    w = np.exp(-np.float64(z[1].abs()))
    want = (LAST * (1 + (V - 1) * w) - 1) / w
    for s in ({}, {"m": 1e-15}, {"k": V - 1}):
        for us in ([LAST], [LAST] * 6):
            got = _check(z, us, **s)
            assert all(abs(x - want) <= 0.01 * V for x in got), (s, got, want)
    assert _check(z, [1.0, 2.0]) == [V - 1] * 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [20011, 131072, (1 << 20) - 5])
@pytest.mark.parametrize("turned", [False, True])
def test_parts_further_and_further_below(turned, V, dtype):
    """Blocks of 3000 tokens, each 4 nats below the one before (behind it), down to 50."""
    g = torch.Generator().manual_seed(V)
    z = -4.0 * (torch.arange(V) // 3000).clamp(max=12).float() + torch.randn(V, generator=g) * 0.5
    z[torch.arange(V) // 3000 >= 13] = -50.0
    z = (z.flip(0) if turned else z).to(dtype)
    for s in SETTINGS:
        s = dict(s)
        if "k" in s:
            s["k"] = 2 * V // 3
        _check(z, **s)


def test_a_last_part_of_one_slice():
    """131072 tokens whose last slice alone lies 34 nats below: a number of 1 draws its last."""
    for dtype in (torch.float32, torch.bfloat16):
        V = 131072
        z = torch.zeros(V)
        z[-8192:] = -34.0
        z[:-8192][1::2] = float("-inf")
        z = z.to(dtype)
        assert _check(z, [1.0, 5.0]) == [V - 1] * 2
        z[-3:] = float("-inf")
        z[-8192:-8000] = float("nan")
        assert _check(torch.where(z.isnan(), -float("inf"), z.float()).to(dtype), [1.0])[0] == V - 4
        got = sample_tokens(_rows(z, 3), torch.tensor([1.0, LAST, 0.0], device=DEV)).tolist()
        assert got[0] == V - 4 and got[1] < V - 8192 and got[2] == 0
