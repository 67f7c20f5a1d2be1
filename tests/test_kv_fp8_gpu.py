"""The 8-bit KV cache's write and read against a plain 64-bit form on the host: codes and
scales bit for bit (the rounding is defined to the last case), bytes that no token goes to
included."""

import pytest
import torch

from evo2_flash_amd.attention import PagedKVCache, rotary_decode, rotary_prefill
from evo2_flash_amd.kv_fp8 import (Fp8KVCache, read_kv_fp8, rotary_decode_fp8, rotary_prefill_fp8,
                                   write_kv_fp8)

from _kv_fp8 import F8, PAGE, random_cache, write_side

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _host(cache):
    k, v, ks, vs = (t.detach().cpu() for t in cache)
    return [k.double(), v.transpose(2, 3).double().contiguous(), ks.double(), vs.double()]


def _same(cache, want):
    k, v, ks, vs = _host(cache)
    for name, a, b in (("k", k, want[0]), ("v", v, want[1]), ("k_scale", ks, want[2]), ("v_scale", vs, want[3])):
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        assert torch.equal(a.nan_to_num(nan=1e9), b.nan_to_num(nan=1e9)), name


def _tokens(B, n, kv, hd, g, wild):
    x = torch.randn(B, n, kv, hd, generator=g) * torch.exp2(
        torch.randint(-3, 4, (B, n, kv, 1), generator=g).float())
    if wild:
        flat = x.view(-1)
        for value in (float("inf"), float("-inf"), float("nan"), 0.0, 3.0e38, 2.0 ** -130, 1.0e-30, 448.0, 452.0):
            at = torch.randint(0, flat.numel(), (3,), generator=g)
            if value < 1e9 or wild == 2:
                flat[at] = value
        x[:, :, 0] = x[:, :, 0] * (1e-38 if wild == 2 else 0.0)
    return x.to(BF)


CASES = [  # starts, lengths (None: n), n
    ([0], None, 1), ([0, 5, 15, 16, 31], None, 1), ([0, 7], None, 16), ([0, 1, 15], None, 17),
    ([3, 16, 0, 40, 2], [40, 0, 17, 1, 33], 40), ([0], None, 700), ([13], [-5], 20), ([30], [99], 2),
]


@pytest.mark.parametrize("wild", [0, 1, 2])
@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 128), (8, 64), (5, 128)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_and_read(case, kv, hd, wild):
    starts, lengths, n = CASES[case]
    B = len(starts)
    g = torch.Generator().manual_seed(1000 * case + 10 * kv + wild)
    cols = max(-(-(a + n) // PAGE) for a in starts) + 1
    pages = B * cols + 2
    table = (torch.randperm(pages - 1, generator=g)[:B * cols] + 1).view(B, cols).to(torch.int32)
    cache = random_cache(pages, kv, hd, g, DEV)
    want = _host(cache)
    k, v = _tokens(B, n, kv, hd, g, wild), _tokens(B, n, kv, hd, g, wild)
    count = [n] * B if lengths is None else [min(max(m, 0), n) for m in lengths]
    write_side(k, want[0], want[2], table, starts, count)
    write_side(v, want[1], want[3], table, starts, count)
    rows = torch.cat([k, v], 2).to(DEV)  # values as a view of the step's rows
    pos = torch.tensor(starts, device=DEV)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    write_kv_fp8(rows[:, :, :kv], rows[:, :, kv:], *cache, table.to(DEV), pos, lens)
    _same(cache, want)
    ends = torch.tensor([a + m for a, m in zip(starts, count)])
    L = int(ends.max()) + 3
    got = read_kv_fp8(*cache, table.to(DEV), ends.to(DEV), L)
    for x, codes, scale in zip(got, want[:2], want[2:]):
        ref = torch.zeros(B, L, kv, hd, dtype=torch.float64)
        for b in range(B):
            at = torch.arange(int(ends[b]))
            pg = table[b].long()[at // PAGE]
            ref[b, :len(at)] = codes[pg, :, at % PAGE] * scale[pg][..., None]
        a = x.cpu().double()
        assert torch.equal(torch.isnan(a), torch.isnan(ref))
        assert torch.equal(a.nan_to_num(nan=1e39), ref.nan_to_num(nan=1e39))


@pytest.mark.parametrize("kv,hd", [(2, 64), (4, 128)])
def test_tokens_one_by_one_that_grow(kv, hd):
    """Each token of a page larger than those before: every write re-encodes."""
    g = torch.Generator().manual_seed(3)
    table = torch.tensor([[2, 1], [3, 4]], dtype=torch.int32)
    cache = random_cache(5, kv, hd, g, DEV)
    want = _host(cache)
    x = _tokens(2, 20, 2 * kv, hd, g, 0) * torch.exp2(0.7 * torch.arange(20.0))[None, :, None, None].to(BF)
    for i in range(20):
        k, v = x[:, i:i + 1, :kv], x[:, i:i + 1, kv:]
        write_side(k, want[0], want[2], table, [i, i + 3], [1, 1])
        write_side(v, want[1], want[3], table, [i, i + 3], [1, 1])
        write_kv_fp8(k.to(DEV), v.to(DEV), *cache, table.to(DEV), torch.tensor([i, i + 3], device=DEV))
        _same(cache, want)


def test_places_outside_the_table_and_the_pages():
    g = torch.Generator().manual_seed(4)
    cache = random_cache(4, 2, 64, g, DEV)
    want = _host(cache)
    table = torch.tensor([[1, -1, 2], [9, 4, 3], [1, 2, 3], [1, 2, 3], [1, 2, 3]], dtype=torch.int32)
    starts = [0, 0, -1, 48, 1 << 40]
    k = _tokens(5, 60, 2, 64, g, 0)
    write_side(k, want[0], want[2], table, starts, [60] * 5)
    write_side(k, want[1], want[3], table, starts, [60] * 5)
    write_kv_fp8(k.to(DEV), k.to(DEV), *cache, table.to(DEV), torch.tensor(starts, device=DEV))
    _same(cache, want)
    got, _ = read_kv_fp8(*cache, table.to(DEV), torch.tensor([60, -3, 1 << 40, 17, 1], device=DEV), 50)
    assert not got[0, 16:32].any() and not got[0, 48:].any() and not got[1].any()
    assert got[0, :16].any() and got[2, 47].any() and not got[2, 48:].any()
    assert not got[3, 17:].any() and not got[4, 1:].any()


def test_views_that_are_copied_and_empty_calls():
    g = torch.Generator().manual_seed(5)
    cache = random_cache(4, 2, 64, g, DEV)
    want = _host(cache)
    table = torch.tensor([[3, 1]], dtype=torch.int32)
    wide = _tokens(1, 21, 2, 65, g, 0)
    k, v = wide[..., 1:], _tokens(1, 21, 64, 2, g, 0).transpose(2, 3)  # unaligned; strided last
    write_side(k, want[0], want[2], table, [2], [21])
    write_side(v, want[1], want[3], table, [2], [21])
    write_kv_fp8(wide.to(DEV)[..., 1:], v.transpose(2, 3).contiguous().to(DEV).transpose(2, 3), *cache,
                 table.to(DEV), torch.tensor([2], dtype=torch.int32, device=DEV))
    _same(cache, want)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    write_kv_fp8(k[:0].to(DEV), v[:0].contiguous().to(DEV), *cache, table.to(DEV), none)
    write_kv_fp8(k[:, :0].to(DEV), v[:, :0].contiguous().to(DEV), *cache, table.to(DEV), none.new_zeros(1))
    _same(cache, want)
    assert read_kv_fp8(*cache, table.to(DEV), none, 5)[0].shape == (0, 5, 2, 64)
    assert read_kv_fp8(*cache, table.to(DEV), none.new_ones(1), 0)[1].shape == (1, 0, 2, 64)


def test_pages_past_32_bit_offsets():
    """A cache of over 4 GB a side, pages further apart than they are long."""
    kv, hd, pages = 2, 128, 40000
    big = [torch.zeros(pages, 29, 2048, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2)]
    k, v = big[0][:, 3:5].view(pages, kv, PAGE, hd), big[1][:, 26:28].view(pages, kv, hd, PAGE)
    scales = [torch.ones(pages, kv, device=DEV) for _ in range(2)]
    table = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(6)
    x = _tokens(1, 41, 2 * kv, hd, g, 0).to(DEV)
    cache = (k, v, *scales)
    write_kv_fp8(x[:, :, :kv], x[:, :, kv:], *cache, table, torch.zeros(1, dtype=torch.int64, device=DEV))
    small = [torch.zeros(4, kv, PAGE, hd, device=DEV).to(F8), torch.zeros(4, kv, hd, PAGE, device=DEV).to(F8),
             torch.ones(4, kv, device=DEV), torch.ones(4, kv, device=DEV)]
    near = torch.tensor([[3, 1, 2]], dtype=torch.int32, device=DEV)
    write_kv_fp8(x[:, :, :kv], x[:, :, kv:], *small, near, torch.zeros(1, dtype=torch.int64, device=DEV))
    ends = torch.tensor([41], device=DEV)
    for a, b in zip(read_kv_fp8(*cache, table, ends, 41), read_kv_fp8(*small, near, ends, 41)):
        assert torch.equal(a, b) and a.any()
    assert not big[0][:pages - 2, 5:].view(torch.uint8)[2:].any()


@pytest.mark.parametrize("hd", [64, 128])
def test_rotary_decode_writes_what_rotary_and_write_do(hd):
    """q's bits are rotary_decode's, the cache's those of its keys and the values written."""
    nh, B = 5, 4
    g = torch.Generator().manual_seed(7)
    table = torch.tensor([[1, 2], [3, 4], [5, -1], [6, 7]], dtype=torch.int32, device=DEV)
    inv = (1.0 / 10000.0 ** (torch.arange(0, hd, 2).float() / hd)).to(DEV)
    plain = PagedKVCache(8, nh, hd, DEV)
    one, two = Fp8KVCache(8, nh, hd, DEV), Fp8KVCache(8, nh, hd, DEV)
    for step in range(20):
        pos = torch.tensor([step, step + 9, step, 31 - step], device=DEV)
        rows = (torch.randn(B, 3 * nh * hd, generator=g) * 1.13 ** step).to(BF).to(DEV)
        if step == 7:
            rows[:, -1] = float("inf")
        q = rotary_decode(rows, plain, table, pos, inv, 4.0)
        assert torch.equal(rotary_decode_fp8(rows, one, table, pos, inv, 4.0), q)
        b = torch.arange(B, device=DEV)
        page = table[b, pos // PAGE].long().clamp(min=0)
        k, v = plain.k[page, :, :, pos % PAGE], plain.v[page, :, pos % PAGE]
        two.append(k, v, table, pos)
        for x, y in zip(one.tensors, two.tensors):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), step


@pytest.mark.parametrize("L", [1, 16, 75, 200])
def test_rotary_prefill_keeps_its_operands(L):
    nh, hd, nseq = 4, 128, 2
    g = torch.Generator().manual_seed(8)
    cols = -(-L // PAGE)
    table = (torch.arange(nseq * cols) + 1).view(nseq, cols).to(torch.int32).to(DEV)
    inv = (1.0 / 10000.0 ** (torch.arange(0, hd, 2).float() / hd)).to(DEV)
    rows = torch.randn(nseq * L, 3 * nh * hd, generator=g).to(BF).to(DEV)
    plain, cache = PagedKVCache(nseq * cols + 1, nh, hd, DEV), Fp8KVCache(nseq * cols + 1, nh, hd, DEV)
    a = rotary_prefill(rows, plain, table, inv, 1.0, nseq, L)
    b = rotary_prefill_fp8(rows, cache, table, inv, 1.0, nseq, L)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    want = Fp8KVCache(nseq * cols + 1, nh, hd, DEV)
    kd, vd = plain.dense(table, nseq, L)
    want.write_prompt(kd.transpose(2, 3), vd, table)
    kq, vq = cache.dense(table, nseq, L)
    for x, y in zip((kq, vq), want.dense(table, nseq, L)):
        assert torch.equal(x, y)
    # a code is off by at most half a step: 2^-4 of the value, or half the subnormal step 2^-9
    # of a scale that is at most 2 max / 448
    for x, y in zip((kq, vq), (kd, vd)):
        x, y = x.double(), y.double()
        assert ((x - y).abs() <= 2.0 ** -4 * y.abs() + 2.0 ** -9 * y.abs().max() / 448).all()
