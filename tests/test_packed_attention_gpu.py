"""attention.packed_attention and its gradients against 64-bit arithmetic.

Bounds (u = 2^-8, half a bf16 step; e = 2^-24): a score is off by es = (hd + 4) e scale
sum |q k| and a probability relatively by twice the row's largest es plus the rounding
of the exponent's argument; as a bf16 operand it is off by u p more.  o is rounded once.
In the backward pass p (dp - delta) is rounded once as an operand, delta from o to 2^-16;
each gradient is rounded once.
"""

import pytest
import torch

from evo2_flash_amd.attention import packed_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
U, E = 2.0 ** -8, 2.0 ** -24


def _case(lens, heads, kv, hd, seed, pad=(0, 0), dev=1.3):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + sum(pad)
    q, k, v, d = ((torch.randn(T, n, hd, generator=g) * dev).to(BF).to(DEV)
                  for n in (heads, kv, kv, heads))
    cu = torch.tensor([pad[0], *lens]).cumsum(0).to(torch.int32).to(DEV)
    return q, k, v, d, cu


def _exact(q, k, v, d, cu, scale):
    """{name: (value, bound)} in 64 bits."""
    q, k, v, d = (t.detach().cpu().double() for t in (q, k, v, d))
    cu = cu.cpu().tolist()
    heads, kv, hd = q.shape[1], k.shape[1], q.shape[2]
    r = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    b = {n: torch.zeros_like(t) for n, t in r.items()}
    for s0, s1 in zip(cu[:-1], cu[1:]):
        n = s1 - s0
        if n <= 0:
            continue
        s = slice(s0, s1)
        live = torch.ones(n, n, dtype=torch.bool).tril()
        for h in range(heads):
            j = h // (heads // kv)
            sc = (q[s, h] @ k[s, j].t()) * scale
            mag = (q[s, h].abs() @ k[s, j].abs().t()) * scale * live
            p = torch.softmax(sc.masked_fill(~live, float("-inf")), 1)
            top = (sc.abs() * live).amax(1, keepdim=True)
            rp = 2 * (hd + 4) * E * mag.amax(1, keepdim=True) + (8 * top + n + 16) * E
            o = p @ v[s, j]
            so = p @ v[s, j].abs()
            eo = (U + rp + (n + 8) * E) * so
            r["o"][s, h] = o
            b["o"][s, h] = U * o.abs() + eo
            dp = d[s, h] @ v[s, j].t()
            sdp = d[s, h].abs() @ v[s, j].abs().t()
            delta = (p * dp).sum(1, keepdim=True)
            # delta = do . o: o to a bf16 pair, whose error is e_o (fp32) + u^2 |o| / 2,
            # the probabilities' own roundings (u p, before the value product) among it
            edelta = (d[s, h].abs() * (eo + U * U * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eds = (U + 2 * rp) * ds.abs() + p * (2 * (hd + 4) * E * sdp + edelta * 1.01)
            if n >= 1:  # a query of one key: exactly 0
                ds[0] = 0.0
                eds[0] = 0.0
            ep = (U + rp) * p
            r["dq"][s, h] = scale * (ds @ k[s, j])
            b["dq"][s, h] = scale * ((eds + n * E * ds.abs()) @ k[s, j].abs())
            r["dk"][s, j] += scale * (ds.t() @ q[s, h])
            b["dk"][s, j] += scale * ((eds + n * E * ds.abs()).t() @ q[s, h].abs())
            r["dv"][s, j] += p.t() @ d[s, h]
            b["dv"][s, j] += (ep + n * E * p).t() @ d[s, h].abs()
    for n in ("dq", "dk", "dv"):
        b[n] = b[n] * 1.01 + U * r[n].abs()
    return {n: (r[n], b[n]) for n in r}


def _check(got, want, what):
    for n, t in got.items():
        v, bound = want[n]
        off = (t.detach().cpu().double() - v).abs()
        assert bool((off <= bound * (1 + 2 * U) + 1e-38).all()), (
            what, n, float((off / (bound + 1e-30)).max()))


def _grads(q, k, v, d, cu, scale):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, cu, scale)
    return dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, d))))


CASES = [
    ([1], 1, 1, 128), ([2], 2, 1, 64), ([1, 1, 1], 8, 8, 64), ([31, 32, 33], 4, 2, 128),
    ([63, 64, 65], 3, 3, 64), ([127, 128, 129], 2, 2, 128), ([5, 0, 7, 0, 0, 200], 4, 1, 128),
    ([257], 8, 8, 128), ([400, 3, 77], 16, 8, 64), ([640], 2, 1, 64), ([1000], 1, 1, 128),
    ([1] * 150 + [3, 70], 2, 2, 64),
]


@pytest.mark.parametrize("lens,heads,kv,hd", CASES)
def test_against_64_bits(lens, heads, kv, hd):
    q, k, v, d, cu = _case(lens, heads, kv, hd, seed=sum(lens) + hd)
    scale = hd ** -0.5
    print(f"packed_attention {lens[:8]} {heads} {kv} {hd}", flush=True)
    want = _exact(q, k, v, d, cu, scale)
    with torch.no_grad():
        _check({"o": packed_attention(q, k, v, cu, scale)}, want, "forward")
    _check(_grads(q, k, v, d, cu, scale), want, "training")


@pytest.mark.parametrize("heads,kv,hd,pad", [(8, 8, 128, (3, 40)), (16, 2, 128, (260, 5)), (6, 3, 128, (0, 1)),
                                             (16, 4, 64, (7, 300))])
def test_enough_workgroups_for_larger_ones(heads, kv, hd, pad):
    """Key tiles of 256 rows, whole, cut short and of one key, behind one another; rows
    outside the sequences cleared by workgroups of that size."""
    lens = [513, 31, 257, 0, 256] + [2, 1] * 30 + [300]
    q, k, v, d, cu = _case(lens, heads, kv, hd, seed=heads + pad[0], pad=pad)
    print(f"packed_attention, larger workgroups {heads} {kv} {hd} {pad}", flush=True)
    _check(_grads(q, k, v, d, cu, hd ** -0.5), _exact(q, k, v, d, cu, hd ** -0.5), "training")


@pytest.mark.parametrize("nseq", [64, 65, 4097])
def test_many_sequences(nseq):
    """Tables of one, two and three search steps, empty sequences among them."""
    g = torch.Generator().manual_seed(nseq)
    lens = torch.randint(0, 4, (nseq,), generator=g).tolist()
    lens[nseq // 2] = 300
    q, k, v, d, cu = _case(lens, 2, 1, 64, seed=nseq, pad=(1, 2))
    print(f"packed_attention, {nseq} sequences", flush=True)
    _check(_grads(q, k, v, d, cu, 0.125), _exact(q, k, v, d, cu, 0.125), "training")


@pytest.mark.parametrize("pad", [(0, 9), (130, 0), (3, 300)])
def test_rows_outside_the_sequences(pad):
    """Rows before the first and behind the last sequence: zeros, and zero gradients,
    whatever they hold."""
    q, k, v, d, cu = _case([70, 1, 33], 4, 2, 128, seed=5, pad=pad)
    out = torch.ones(q.shape[0], dtype=torch.bool)
    out[pad[0]:q.shape[0] - pad[1]] = False
    for t in (q, k, v, d):
        t[out.to(DEV)] = float("nan")
    got = _grads(q, k, v, d, cu, 0.09)
    for t in (q, k, v, d):
        t[out.to(DEV)] = 0.0
    want = _exact(q, k, v, d, cu, 0.09)
    _check(got, want, pad)
    for n, t in got.items():
        assert not t[out.to(DEV)].any(), n


def test_gradient_against_differences():
    """The output is linear in v: along a direction exact in bf16 the difference is the
    gradient but for the outputs' roundings.  In q and k along a small direction, the
    second order below the roundings."""
    q, k, v, d, cu = _case([40, 1, 90], 4, 2, 64, seed=21)
    got = _grads(q, k, v, d, cu, 0.125)
    g = torch.Generator().manual_seed(22)
    for i, (n, size) in enumerate((("dq", 2.0 ** -4), ("dk", 2.0 ** -4), ("dv", 0.5))):
        ops = [q, k, v]
        step = (torch.randint(0, 2, ops[i].shape, generator=g) * 2 - 1).to(DEV) * size
        lo, hi = ((ops[i].float() + s * step).to(BF) for s in (-1, 1))
        with torch.no_grad():
            a, b = (packed_attention(*ops[:i], t, *ops[i + 1:], cu, 0.125).double() for t in (lo, hi))
        want = ((b - a) * d.double()).sum()
        have = (got[n].double() * (hi.double() - lo.double())).sum()
        noise = U * ((a.abs() + b.abs()) * d.double().abs()).square().sum().sqrt()
        # third order: (0.125 sum |step| |k|)^3 / 6 of the values, some 0.1 of a step's
        third = 0.0 if n == "dv" else 0.02 * noise / U * size
        assert abs(have - want) <= 4 * noise + third, (n, have.item(), want.item())


def test_one_key_rows_have_no_score_gradient():
    """Sequences of one token: out = v, dv = do, dq and dk exactly 0 (also of scores far
    from 0)."""
    q, k, v, d, cu = _case([1] * 9, 4, 4, 128, seed=23, dev=30.0)
    got = _grads(q, k, v, d, cu, 1.0)
    assert torch.equal(got["o"], v) and torch.equal(got["dv"], d)
    assert not got["dq"].any() and not got["dk"].any()


def test_large_scores():
    """Scores of some +-4000: probabilities of 0 and 1 without overflow, the neighbours'
    rows untouched by a sequence of infinities."""
    q, k, v, d, cu = _case([70, 65, 130], 2, 1, 128, seed=24)
    want = _grads(q, k, v, d, cu, 0.09)
    big = _grads(q * 32, k * 32, v, d, cu, 0.09)
    assert all(t.isfinite().all() for t in big.values())
    for t in (q, k, v):
        t[70:135] = float("inf")
    got = _grads(q, k, v, d, cu, 0.09)
    for n in want:
        assert torch.equal(got[n][:70], want[n][:70]) and torch.equal(got[n][135:], want[n][135:]), n


def test_forms_of_call():
    """Views of the projection's rows, unaligned and expanded operands, int64 lengths, one
    gradient asked for, no rows, no sequences: the same values."""
    lens, heads, kv, hd = [50, 7, 140], 4, 2, 64
    q, k, v, d, cu = _case(lens, heads, kv, hd, seed=25)
    T = sum(lens)
    want = _grads(q, k, v, d, cu, 0.1)
    rows = torch.zeros(T, (heads + 2 * kv) * hd + 24, dtype=BF, device=DEV)
    rows[:, 8:-16] = torch.cat([t.reshape(T, -1) for t in (q, k, v)], 1)
    qv, kvw, vv = rows[:, 8:-16].view(T, heads + 2 * kv, hd).split([heads, kv, kv], 1)
    assert qv.data_ptr() % 16 == 0 and not qv.is_contiguous()
    got = _grads(qv, kvw, vv, d.transpose(0, 1).contiguous().transpose(0, 1), cu.long(), 0.1)
    assert all(torch.equal(got[n], want[n]) for n in want)
    odd = torch.zeros(T * heads * hd + 1, dtype=BF, device=DEV)[1:].view(T, heads, hd).copy_(q)
    assert torch.equal(packed_attention(odd, k, v, cu, 0.1), want["o"])
    # a key head expanded over the query heads equals sharing it
    ke, ve = (t[:, :1].expand(T, heads, hd) for t in (k, v))
    assert torch.equal(packed_attention(q, ke, ve, cu, 0.1),
                       packed_attention(q, k[:, :1], v[:, :1], cu, 0.1))
    qs = q.clone().requires_grad_()
    packed_attention(qs, k, v, cu, 0.1).sum().backward()
    assert torch.equal(qs.grad, _grads(q, k, v, torch.ones_like(d), cu, 0.1)["dq"])
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _grads(q, k, v, d, none, 0.1)  # no sequences: every row is outside
    assert not any(t.any() for t in got.values())
    assert packed_attention(q[:0], k[:0], v[:0], none, 0.1).shape == (0, heads, hd)


def test_lengths_that_lie_outside():
    """Entries past the rows are clamped: nothing outside is read or written."""
    q, k, v, d, cu = _case([100, 60], 2, 2, 64, seed=26)
    far = cu.clone()
    far[-1], far[0] = 100000, -7
    want, got = _grads(q, k, v, d, cu, 0.1), _grads(q, k, v, d, far, 0.1)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2)])
def test_repeats_bit_for_bit_in_a_graph(heads, kv):
    """Replays of a captured forward and backward pass, with eager work between, give the
    eager bits; so does another stream."""
    q, k, v, d, cu = _case([200, 33, 64], heads, kv, 128, seed=27)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        o = packed_attention(*leaves, cu, 0.1)
        return (o.detach(), *torch.autograd.grad(o, leaves, d))

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    want = _grads(q, k, v, d, cu, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(first, want.values()))
    for rep in range(3):
        with torch.no_grad():
            leaves[2].copy_(v * (rep + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = _grads(q, k, v * (rep + 1), d, cu, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager.values())), rep
