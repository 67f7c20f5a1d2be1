"""Decode attention over the 8-bit cache against 64-bit attention of the values its codes
stand for.

Tolerance, from the arithmetic: the operands are exact, a score is an fp32 sum of head_dim
exact products (error below head_dim 2^-24 of the sum of their magnitudes, whose largest is
`worst`), a probability carries twice that as a relative error (its own and its row's sum's)
besides the bf16 pair's 2^-16 and the sums over positions' and the exponentials' few 2^-24;
the result is rounded to bf16 once (half a step, 2^-8 of it)."""

import pytest
import torch

from evo2_flash_amd.kv_fp8 import (Fp8KVCache, paged_decode_attention_fp8, workspace_fp8, write_kv_fp8)

from _kv_fp8 import PAGE, attention_exact, random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _check(out, q, cache, table, positions, scale):
    ref, mass, worst = attention_exact(q, *[t.cpu() for t in cache], table, positions, scale)
    hd, L = q.shape[-1], table.shape[1] * PAGE
    rel = 2 * hd * 2.0 ** -24 * worst + 2.0 ** -16 + (L + 64) * 2.0 ** -24
    err = (out.cpu().double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + rel * mass * (1 + 2.0 ** -8)).all(), float(
        (err - 2.0 ** -8 * ref.abs() - rel * mass).max())


def _case(lens, n, heads, kv, hd, seed, shared=0, cols=0):
    """Random codes in a table whose unused entries name no page."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-(m + n - 1) // PAGE) - shared) for m in lens]
    cols = max(cols, shared + max(need), 1)
    pages = shared + sum(need) + 2
    perm = (torch.randperm(pages - 1, generator=g) + 1).to(torch.int32)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    table[:, :shared] = perm[:shared]
    at = shared
    for b, m in enumerate(need):
        table[b, shared:shared + m] = perm[at:at + m]
        at += m
    k, v, ks, vs = random_cache(pages, kv, hd, g, DEV)
    # scales that keep scores within some tens and differ by page
    ks *= 2.0 ** -9
    vs *= 2.0 ** -6
    q = torch.randn(len(lens), n, heads, hd, generator=g).to(BF)
    return q, (k, v, ks, vs), table, [m - 1 for m in lens]


SHAPES = [  # lens (the first token's), n, heads, kv, hd
    ([1], 1, 1, 1, 64), ([1, 2, 15, 16, 17, 63, 64, 65], 1, 4, 4, 128), ([0, 5, 0, 130], 1, 2, 2, 64),
    ([255, 256, 257, 511, 513, 1], 1, 8, 2, 128), ([777], 1, 32, 32, 128), ([2047, 2048, 2049, 4097], 1, 2, 1, 64),
    ([1, 16, 100, 255], 3, 6, 2, 128), ([1, 300, 15], 5, 16, 2, 64), ([40, 77], 7, 20, 1, 128),
    ([3000], 2, 24, 1, 64), ([6001, 3, 1500], 1, 3, 3, 128),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_against_64_bits(shape):
    lens, n, heads, kv, hd = SHAPES[shape]
    q, cache, table, pos = _case(lens, n, heads, kv, hd, shape)
    args = (*cache, table.to(DEV), torch.tensor(pos, device=DEV), hd ** -0.5)
    out = paged_decode_attention_fp8(q.to(DEV), *args)
    _check(out, q, cache, table, pos, hd ** -0.5)
    if n == 1:
        assert torch.equal(paged_decode_attention_fp8(q[:, 0].to(DEV), *args), out[:, 0])


@pytest.mark.parametrize("cols", [1, 16, 17, 400, 5000])
def test_tables_longer_than_the_sequences(cols):
    """The split goes by the table: results stay within the tolerance whatever it is."""
    q, cache, table, pos = _case([5, 16, 11], 1, 4, 2, 128, 50, cols=cols)
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), 0.1)
    _check(out, q, cache, table, pos, 0.1)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_chunks_of_waves(shape):
    """A table too long for a workgroup to a sequence: the same calls in joined chunks."""
    lens, n, heads, kv, hd = SHAPES[shape]
    q, cache, table, pos = _case(lens, n, heads, kv, hd, shape, cols=2100)
    work = workspace_fp8(len(lens), heads, kv, hd, 2100, DEV, n=n)
    assert work.numel() > 16
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), hd ** -0.5, work=work)
    _check(out, q, cache, table, pos, hd ** -0.5)


@pytest.mark.parametrize("B,kv,hd", [(64, 4, 128), (37, 7, 64), (1, 1, 64), (2, 128, 128)])
def test_a_workgroup_to_a_sequence(B, kv, hd):
    """Around as many workgroups as CUs, ragged lengths, none of a workspace needed."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 700, (B,), generator=g).tolist()
    q, cache, table, pos = _case(lens, 1, kv, kv, hd, 60 + B)
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), hd ** -0.5,
                                     work=torch.empty(0, device=DEV) if B in (1, 2, 64) else None)
    _check(out, q, cache, table, pos, hd ** -0.5)


@pytest.mark.parametrize("B,shared,n,heads,kv,hd", [(3, 17, 1, 4, 4, 128), (33, 40, 1, 2, 2, 64),
                                                    (5, 129, 2, 8, 2, 128), (40, 64, 1, 2, 1, 128)])
def test_shared_pages(B, shared, n, heads, kv, hd):
    lens = [shared * PAGE + 1 + 7 * (b % 9) for b in range(B)]
    lens[1] = 100  # ends inside the shared pages
    q, cache, table, pos = _case(lens, n, heads, kv, hd, 70 + B, shared=shared)
    args = (*cache, table.to(DEV), torch.tensor(pos, device=DEV), hd ** -0.5)
    for declared in (shared, shared // 2, 0):
        out = paged_decode_attention_fp8(q.to(DEV), *args, shared_pages=declared)
        _check(out, q, cache, table, pos, hd ** -0.5)


def test_entries_outside_the_pages_and_bytes_behind_the_end():
    """Masked pages are left out, a row of nothing else gives zeros; NaN codes behind the
    last position and in page 0 do not reach the result."""
    q, cache, table, pos = _case([70, 33, 200, 9], 1, 4, 2, 64, 90)
    table[0, 1], table[1, 0], table[2, 3] = -1, 1 << 30, cache[0].shape[0]
    table[3, 0] = -7
    for t in cache[:2]:
        t.view(torch.uint8)[0] = 0x7F
    k8, v8 = (t.view(torch.uint8) for t in cache[:2])
    for b, p in enumerate(pos):
        pg = int(table[b, p // PAGE])
        if 0 <= pg < k8.shape[0] and p % PAGE < 15:
            k8[pg, :, p % PAGE + 1:] = 0xFF
            v8[pg, :, :, p % PAGE + 1:] = 0x7F
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), 0.125)
    assert torch.isfinite(out).all() and not out[3].any()
    _check(out, q, cache, table, pos, 0.125)


def test_nan_and_infinite_values_that_are_attended_to():
    q, cache, table, pos = _case([40, 40], 1, 2, 2, 64, 91)
    cache[1].view(torch.uint8)[int(table[0, 1]), 1, 5, 3] = 0x7F
    cache[0].view(torch.uint8)[int(table[1, 0]), 0, 2, 9] = 0x7F
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), 0.125).cpu()
    nan = torch.isnan(out)
    assert nan[0, 0, 1, 5] and nan[0].sum() == 1          # a value's dim
    assert nan[1, 0, 0].all() and nan[1].sum() == 64      # a key's whole head


@pytest.mark.parametrize("hd,shared,cols", [(64, 0, 0), (128, 0, 0), (64, 4, 0), (128, 4, 0), (64, 0, 2100), (128, 0, 2100)])
def test_nan_values_reach_the_tokens_that_attend_to_them(hd, shared, cols):
    """Later tokens of a sequence, or sequences that end further on in shared pages, attend to
    NaN codes that the others do not: theirs alone are NaN, in those dims alone."""
    n, lens = (5, [28, 1, 62]) if not shared else (1, [20, 70, 33, 64, 40])
    q, cache, table, pos = _case(lens, n, 4, 2, hd, 93, shared=shared, cols=cols)
    v8 = cache[1].view(torch.uint8)
    bad = [(0, 30, 0, 3), (0, 31, 1, 60), (1, 2, 0, 9), (2, 64, 1, 17)] if not shared else [
        (0, 25, 0, 3), (0, 39, 0, 40), (0, 63, 1, 5), (0, 19, 1, 33)]
    for b, l, j, d in bad:
        v8[int(table[b, l // PAGE]), j, d, l % PAGE] = 0x7F if d % 2 else 0xFF
    out = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), 0.125,
                                     shared_pages=shared).cpu()
    want = torch.zeros(out.shape, dtype=torch.bool)
    for b, l, j, d in bad:
        for s in (range(len(lens)) if shared else [b]):
            for i in range(n):
                if l <= pos[s] + i:
                    want[s, i, 2 * j:2 * j + 2, d] = True
    assert torch.equal(torch.isnan(out), want)
    for b, l, j, d in bad:
        v8[int(table[b, l // PAGE]), j, d, l % PAGE] = 0
    clean = paged_decode_attention_fp8(q.to(DEV), *cache, table.to(DEV), torch.tensor(pos, device=DEV), 0.125,
                                       shared_pages=shared).cpu()
    assert torch.equal(out[~want], clean[~want])


@pytest.mark.parametrize("cols", [0, 2100])
def test_strides_workspace_and_streams(cols):
    q, cache, table, pos = _case([300, 1000, 17], 2, 8, 4, 128, 92, cols=cols)
    d = (table.to(DEV), torch.tensor(pos, dtype=torch.int32, device=DEV), 0.09)
    want = paged_decode_attention_fp8(q.to(DEV), *cache, *d)
    wide = torch.zeros(3, 2, 8, 200, dtype=BF, device=DEV)
    wide[..., 3:131] = q.to(DEV)
    work = workspace_fp8(8, 8, 4, 128, table.shape[1], DEV, n=2)
    assert torch.equal(paged_decode_attention_fp8(wide[..., 3:131], *cache, *d, work=work), want)
    flat = q.to(DEV).permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)
    assert torch.equal(paged_decode_attention_fp8(flat, *cache, *d, work=work), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged_decode_attention_fp8(q.to(DEV), *cache, *d)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    # pages of a larger pool: heads and pages apart
    k, v, ks, vs = cache
    pool = torch.zeros(k.shape[0], 9, 2048, dtype=torch.uint8, device=DEV)
    pool[:, 0:8:2] = k.view(torch.uint8).view(-1, 4, 2048)
    pool[:, 1:9:2] = v.view(torch.uint8).view(-1, 4, 2048)
    kk = pool[:, 0:8:2].view(k.dtype).unflatten(2, (16, 128))
    vv = pool[:, 1:9:2].view(k.dtype).unflatten(2, (128, 16))
    both = torch.stack([ks, vs], 2)
    assert torch.equal(paged_decode_attention_fp8(q.to(DEV), kk, vv, both[..., 0], both[..., 1], *d), want)


def test_pages_past_32_bit_offsets():
    kv, hd, pages = 2, 128, 40000
    big = [torch.zeros(pages, 29, 2048, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    cache = (big[0][:, 3:5].view(pages, kv, PAGE, hd), big[1][:, 26:28].view(pages, kv, hd, PAGE),
             torch.ones(pages, kv, device=DEV), torch.ones(pages, kv, device=DEV))
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, 41, 2 * kv, hd, generator=g).to(BF).to(DEV)
    q = torch.randn(1, 1, 4, hd, generator=g).to(BF).to(DEV)
    zero, pos = torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([40], device=DEV)
    far = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device=DEV)
    write_kv_fp8(x[:, :, :kv], x[:, :, kv:], *cache, far, zero)
    near = Fp8KVCache(4, kv, hd, DEV)
    table = torch.tensor([[3, 1, 2]], dtype=torch.int32, device=DEV)
    write_kv_fp8(x[:, :, :kv], x[:, :, kv:], *near.tensors, table, zero)
    assert torch.equal(paged_decode_attention_fp8(q, *cache, far, pos, 0.1),
                       paged_decode_attention_fp8(q, *near.tensors, table, pos, 0.1))


@pytest.mark.parametrize("cols", [4, 2100])
def test_decode_step_in_a_graph(cols):
    """Write and attention of a step captured once; each replay against eager calls on
    another cache, with eager work between."""
    B, heads, hd = 3, 4, 64
    table = torch.zeros(B, cols, dtype=torch.int32, device=DEV)
    table[:, :4] = (torch.arange(12, device=DEV) + 1).view(B, 4)
    a, b = Fp8KVCache(13, heads, hd, DEV), Fp8KVCache(13, heads, hd, DEV)
    k, v, q = (torch.zeros(B, heads, hd, dtype=BF, device=DEV) for _ in range(3))
    pos = torch.zeros(B, dtype=torch.int64, device=DEV)
    work = workspace_fp8(B, heads, heads, hd, cols, DEV)

    def step(cache):
        cache.append(k, v, table, pos)
        return paged_decode_attention_fp8(q, *cache.tensors, table, pos, 0.125, work=work)

    step(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    for x, y in zip(a.tensors, b.tensors):  # both as new: the warm-up wrote to one
        x.view(torch.uint8).copy_(y.view(torch.uint8))
    g = torch.Generator().manual_seed(10)
    for i in range(40):
        for t in (k, v, q):
            t.copy_(torch.randn(B, heads, hd, generator=g).to(BF))
        pos.copy_(torch.tensor([i, i + 5, (i + 17) % 64]))
        want = step(b)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want), i
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.tensors, b.tensors))
