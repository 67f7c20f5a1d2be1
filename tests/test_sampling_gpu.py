"""sample_tokens against a plain 64-bit form on the host: the same token everywhere.  (The
kernel's weights are whole numbers of 2^-49 of the largest, over 8192 tokens of 2^-62 V with V
rounded up to a power of two; the reference's are 64-bit; a draw where these would differ lies within some 1e-12 of a border
and does not occur among the seeds here.)"""

import math

import pytest
import torch

from evo2_flash_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _one(z, u, t, k, p, m):
    f = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
    u, t, p, m = f(u), f(t), f(p), f(m)
    z = [float(x) for x in z.double()]
    order = sorted((i for i in range(len(z)) if z[i] > -math.inf), key=lambda i: (-z[i], i))
    if not order:
        return -1
    top = z[order[0]]
    if not t > 0 or k == 1:
        return order[0]
    w = {i: 1.0 if z[i] == top else math.exp((z[i] - top) / t) for i in order}
    if k > 0:
        order = order[:k]
    if p < 1:
        total, run, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and run >= p * total:
                break
            kept.append(i)
            run += w[i]
        order = kept
    order = sorted(i for i in order if w[i] >= min(m, 1.0))
    total, run = math.fsum(w[i] for i in order), 0.0
    for i in order:
        run += w[i]
        if run > u * total:
            return i
    return max(i for i in order if w[i] > 0)


def _check(z, u, t=1.0, k=0, p=1.0, m=0.0):
    B = z.shape[0]
    at = lambda x, b: float(x[b]) if torch.is_tensor(x) else x  # noqa: E731
    want = [_one(z[b], float(u[b]), at(t, b), int(at(k, b)), at(p, b), at(m, b)) for b in range(B)]
    dev = lambda x: x.to(DEV) if torch.is_tensor(x) else x  # noqa: E731
    got = sample_tokens(z.to(DEV), u.to(DEV), dev(t), dev(k), dev(p), dev(m))
    assert got.dtype == torch.int64 and got.tolist() == want


SETTINGS = [(1.0, 0, 1.0, 0.0), (1.0, 4, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 50, 0.95, 0.0), (0.8, 0, 1.0, 0.1),
            (0.5, 20, 0.8, 0.05), (0.0, 3, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (2.0, 0, 0.3, 0.5), (1.0, 10 ** 6, 0.999, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 509, 512, 1025, 4096, 4097, 8192, 8193, 20011, 65537])
def test_settings(V, dtype):
    g = torch.Generator().manual_seed(V)
    for n, (t, k, p, m) in enumerate(SETTINGS):
        z = (torch.randn(5, V, generator=g) * 3).to(dtype)
        _check(z, torch.rand(5, generator=g), t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_longest_rows(dtype):
    V = 1 << 20
    g = torch.Generator().manual_seed(8)
    z = (torch.randn(1, V, generator=g) * 2).to(dtype)
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.9, 70000, 0.8, 0.01)):
        _check(z, torch.rand(1, generator=g), t, k, p, m)


@pytest.mark.parametrize("B,V,dtype", [(350, 8195, torch.bfloat16), (521, 4099, torch.float32)])
def test_many_long_rows(B, V, dtype):
    """Enough rows for slices of 8192: ordinary ones, few values, equal values, masked ones."""
    g = torch.Generator().manual_seed(B)
    z = torch.randn(B, V, generator=g) * 3
    z[::7] = torch.randint(-2, 3, (len(z[::7]), V), generator=g).float()
    z[1::9] = 0.5
    z[2::11, : V - 5] = float("-inf")
    z[3] = float("nan")
    z[4, 40:50] = float("inf")
    pick = lambda v: torch.tensor(v)[torch.randint(len(v), (B,), generator=g)]  # noqa: E731
    _check(z.to(dtype), torch.rand(B, generator=g), pick([0.0, 0.6, 1.0, 1.7]), pick([0, 0, 1, 40, 4096, 5000]),
           pick([0.1, 0.5, 0.95, 1.0]), pick([0.0, 0.0, 0.02, 1.0]))


def test_many_rows():
    g = torch.Generator().manual_seed(9)
    z = torch.randn(70001, 3, generator=g)
    _check(z, torch.rand(70001, generator=g), 0.8, 2, 0.9)


def test_settings_by_row():
    g = torch.Generator().manual_seed(1)
    B, V = 300, 777
    z = torch.randn(B, V, generator=g) * 2
    pick = lambda v: torch.tensor(v)[torch.randint(len(v), (B,), generator=g)]  # noqa: E731
    _check(z, torch.rand(B, generator=g), pick([0.0, 0.5, 1.0, 1.7]), pick([0, 1, 3, 40, 5000]),
           pick([0.1, 0.5, 0.95, 1.0]), pick([0.0, 0.02, 0.5, 1.0]))
    _check(z, torch.rand(B, generator=g), pick([0.5, 1.0]).double(), pick([0, 3, 40]).int(), 0.9, pick([0.0, 0.1]).bfloat16().float())


def test_equal_logits_go_by_index():
    """Ties at the cuts: few values among many tokens, -0 equal to 0."""
    g = torch.Generator().manual_seed(2)
    for V in (40, 512, 3000, 9000):
        z = torch.randint(-2, 3, (40, V), generator=g).float()
        z[z == 0] *= torch.where(torch.rand(int((z == 0).sum()), generator=g) < 0.5, -1.0, 1.0)
        for t, k, p, m in ((1.0, 7, 1.0, 0.0), (1.0, V // 3, 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, V // 2, 0.61, 0.0),
                           (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.3)):
            _check(z, torch.rand(40, generator=g), t, k, p, m)
        same = torch.full((8, V), 1.5)
        u = torch.arange(8) / 8.0
        _check(same, u)
        _check(same, u, 1.0, 0, 0.5)
        _check(same, u, 1.0, 3)


@pytest.mark.parametrize("V", [33, 512, 2000, 6000, 9500])
def test_masked_infinite_and_nan_logits(V):
    g = torch.Generator().manual_seed(3)
    z = torch.randn(12, V, generator=g)
    z[0] = float("-inf")                       # nothing is left
    z[1] = float("nan")
    z[2] = torch.finfo(torch.float32).min      # masked with the lowest value: all equal
    z[3, 1:] = float("-inf")                   # one token
    z[4, ::2] = float("-inf")
    z[5, 5:9] = float("inf")                   # the finite ones have no weight
    z[6, ::3] = float("nan")
    z[7, 3:] = torch.finfo(torch.float32).min  # next to ordinary ones
    z[8] = 3.0e38
    z[8, 7] = -3.0e38
    z[9, :] = float("inf")
    z[10] *= 1e-42
    for t, k, p, m in SETTINGS:
        _check(z, torch.rand(12, generator=g), t, k, p, m)


def test_uniforms_at_and_past_the_ends():
    g = torch.Generator().manual_seed(4)
    for V in (100, 5000, 9000):
        z = torch.randn(7, V, generator=g)
        z[:, 0] = z[:, -1] = float("-inf")
        u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, float("inf"), float("nan")])
        got = sample_tokens(z.to(DEV), u.to(DEV)).tolist()
        assert got == [1, V - 2, V - 2, V - 2, 1, V - 2, 1]


def test_extreme_settings():
    g = torch.Generator().manual_seed(5)
    z = torch.randn(9, 300, generator=g)
    u = torch.rand(9, generator=g)
    first = z.argmax(1).tolist()
    for kw in ({"temperature": 1e-30}, {"top_p": 0.0}, {"top_p": -1.0}, {"min_p": 1.0}, {"min_p": 9.0}, {"temperature": float("nan")},
               {"temperature": -1.0}, {"top_k": 1, "temperature": 5.0}):
        assert sample_tokens(z.to(DEV), u.to(DEV), **kw).tolist() == first, kw
    flat = sample_tokens(z.to(DEV), u.to(DEV), temperature=float("inf")).tolist()
    assert flat == [int(300 * x) for x in u.double()]
    whole = sample_tokens(z.to(DEV), u.to(DEV)).tolist()
    for kw in ({"top_k": -3}, {"top_k": 300}, {"top_p": 1.5}, {"min_p": -1.0}):
        assert sample_tokens(z.to(DEV), u.to(DEV), **kw).tolist() == whole, kw


def test_rows_apart_streams_and_graphs():
    g = torch.Generator().manual_seed(6)
    for V in (500, 4000, 30000):
        wide = torch.randn(6, V + 13, generator=g).to(DEV)
        z, u = wide[:, 5:V + 5], torch.rand(6, generator=g).to(DEV)
        want = sample_tokens(z.contiguous(), u, 0.9, 40, 0.9)
        assert torch.equal(sample_tokens(z, u, 0.9, 40, 0.9), want)
        assert torch.equal(sample_tokens(z.t().contiguous().t(), u, 0.9, 40, 0.9), want)
        assert torch.equal(sample_tokens(z[:1].expand(6, V), u, 0.9, 40, 0.9),
                           sample_tokens(z[:1].repeat(6, 1), u, 0.9, 40, 0.9))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = sample_tokens(z, u, 0.9, 40, 0.9)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        zs, us = z.contiguous(), u.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sample_tokens(zs, us, 0.9, 40, 0.9, 0.01)
        for _ in range(4):
            zs.copy_(torch.randn(6, V, generator=g))
            us.copy_(torch.rand(6, generator=g))
            want = sample_tokens(zs, us, 0.9, 40, 0.9, 0.01)
            torch.cuda.synchronize()
            graph.replay()
            assert torch.equal(out, want)


def test_frequencies():
    """Evenly spaced numbers draw each token as often as its probability says, to one."""
    n = 4096
    z = torch.tensor([[0.0, 1.0, -0.5, 2.0, 0.3]])
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(sample_tokens(z.expand(n, 5).to(DEV), u.to(DEV), 0.8).cpu(), minlength=5)
    want = torch.softmax(z[0].double() / float(torch.tensor(0.8)), 0) * n
    assert ((got - want).abs() <= 1.0).all()


def test_no_rows():
    assert sample_tokens(torch.zeros(0, 7, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)
