"""What the 8-bit cache's operators and the draw refuse, without a GPU: the wrappers' checks
on CPU tensors (the device check apart), the C entries' argument checks, which come before
any launch, and the workspace queries."""

import pytest
import torch

from evo2_flash_amd import _lib
from evo2_flash_amd.kv_fp8 import (Fp8KVCache, paged_decode_attention_fp8, read_kv_fp8, rotary_decode_fp8,
                                   rotary_prefill_fp8, write_kv_fp8)
from evo2_flash_amd.sampling import sample_tokens

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _cache(pages=5, kv=2, hd=64):
    return [torch.zeros(pages, kv, 16, hd, dtype=torch.uint8).view(F8),
            torch.zeros(pages, kv, hd, 16, dtype=torch.uint8).view(F8), torch.ones(pages, kv), torch.ones(pages, kv)]


TABLE = torch.zeros(3, 4, dtype=torch.int32)
POS = torch.zeros(3, dtype=torch.int64)


def test_cpu_tensors_are_refused():
    c = _cache()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        write_kv_fp8(_z(3, 1, 2, 64), _z(3, 1, 2, 64), *c, TABLE, POS)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        read_kv_fp8(*c, TABLE, POS, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_decode_attention_fp8(_z(3, 4, 64), *c, TABLE, POS, 0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        sample_tokens(_z(2, 9), torch.zeros(2))
    cache = Fp8KVCache(3, 2, 64, "cpu")
    for call in (lambda: rotary_decode_fp8(_z(3, 384), cache, TABLE, POS, torch.zeros(32), 1.0),
                 lambda: rotary_prefill_fp8(_z(3, 384), cache, TABLE, torch.zeros(32), 1.0, 1, 3)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.fixture
def native(monkeypatch):
    """CPU tensors pass the device check; a call is an error."""
    def call(name, *args):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "call", call)


def _bad_cache(i, t):
    c = _cache()
    c[i] = t
    return c


BAD_CACHES = [
    (_bad_cache(0, _z(5, 2, 16, 64)), TABLE, "float8_e4m3fn"),
    (_bad_cache(1, torch.zeros(5, 2, 64, 16, dtype=torch.uint8)), TABLE, "float8_e4m3fn"),
    (_bad_cache(0, _cache()[0][..., :8, :]), TABLE, "float8_e4m3fn"),
    (_bad_cache(1, _cache(kv=3)[1]), TABLE, "do not match"),
    (_bad_cache(1, _cache()[0]), TABLE, "do not match"),
    (_cache(hd=80), TABLE, "head_dim 64 or 128"),
    (_bad_cache(2, torch.ones(5, 3)), TABLE, "scales must be"),
    (_bad_cache(3, torch.ones(5, 2, dtype=torch.float64)), TABLE, "scales must be"),
    (_cache(pages=0), TABLE, "no pages"),
    (_cache(kv=0), TABLE, "no pages"),
    (_bad_cache(0, _cache(hd=128)[0].view(torch.uint8)[..., ::2].view(F8)), TABLE, "contiguous"),
    (_bad_cache(1, _cache()[0].view(torch.uint8).transpose(2, 3).view(F8)), TABLE, "contiguous"),
    (_cache(), TABLE.long(), "block_table"),
    (_cache(), TABLE[:2], "block_table"),
    (_cache(), TABLE[:, :0], "block_table"),
    (_cache(), TABLE[0], "block_table"),
    (_cache(), torch.zeros(3, 8, dtype=torch.int32)[:, ::2], "unit column stride"),
]


@pytest.mark.parametrize("i", range(len(BAD_CACHES)))
def test_caches_that_are_refused(native, i):
    c, table, match = BAD_CACHES[i]
    kv, hd = c[0].shape[1], c[0].shape[3]
    with pytest.raises(ValueError, match=match):
        write_kv_fp8(_z(3, 1, kv, hd), _z(3, 1, kv, hd), *c, table, POS)
    with pytest.raises(ValueError, match=match):
        read_kv_fp8(*c, table, POS, 4)
    with pytest.raises(ValueError, match=match):
        paged_decode_attention_fp8(_z(3, max(kv, 1), hd), *c, table, POS, 0.1)


@pytest.mark.parametrize("k,v,pos,lens,match", [
    (_z(3, 2, 64), _z(3, 2, 64), POS, None, "takes bf16 k and v"),
    (_z(3, 1, 2, 64, dtype=torch.float16), _z(3, 1, 2, 64), POS, None, "takes bf16 k and v"),
    (_z(3, 1, 2, 64), _z(3, 2, 2, 64), POS, None, "takes bf16 k and v"),
    (_z(3, 1, 3, 64), _z(3, 1, 3, 64), POS, None, "tokens of"),
    (_z(3, 1, 2, 128), _z(3, 1, 2, 128), POS, None, "tokens of"),
    (_z(4, 1, 2, 64), _z(4, 1, 2, 64), POS, None, "block_table"),
    (_z(3, 1, 2, 64), _z(3, 1, 2, 64), POS[:2], None, "positions must be"),
    (_z(3, 1, 2, 64), _z(3, 1, 2, 64), POS.float(), None, "positions must be"),
    (_z(3, 1, 2, 64), _z(3, 1, 2, 64), POS, POS[None], "lengths must be"),
    (_z(3, 1, 2, 64), _z(3, 1, 2, 64), POS, POS.bool(), "lengths must be"),
])
def test_writes_that_are_refused(native, k, v, pos, lens, match):
    with pytest.raises(ValueError, match=match):
        write_kv_fp8(k, v, *_cache(), TABLE, pos, lens)


def test_reads_that_are_refused(native):
    for lens, L, match in ((POS.float(), 4, "lengths must be"), (POS, -1, "L >= 0"), (POS.view(3, 1), 4, "lengths"),
                           (torch.zeros(4, dtype=torch.int64), 4, "block_table")):
        with pytest.raises(ValueError, match=match):
            read_kv_fp8(*_cache(), TABLE, lens, L)


@pytest.mark.parametrize("q,pos,kw,match", [
    (_z(3, 64), POS, {}, "takes bf16 q"),
    (_z(3, 1, 1, 4, 64), POS, {}, "takes bf16 q"),
    (_z(3, 4, 64, dtype=torch.float32), POS, {}, "takes bf16 q"),
    (_z(3, 4, 128), POS, {}, "does not match pages"),
    (_z(3, 3, 64), POS, {}, "does not match pages"),
    (_z(3, 0, 64), POS, {}, "does not match pages"),
    (_z(3, 4, 64), POS[:1], {}, "positions must be"),
    (_z(3, 4, 64), POS, {"scale": 0.0}, "positive scale"),
    (_z(3, 4, 64), POS, {"scale": float("nan")}, "positive scale"),
    (_z(3, 4, 64), POS, {"scale": float("inf")}, "positive scale"),
    (_z(3, 4, 64), POS, {"shared_pages": 5}, "shared_pages"),
    (_z(3, 4, 64), POS, {"shared_pages": -1}, "shared_pages"),
    (_z(3, 4, 64), POS, {"work": torch.zeros(64, 2)[:, 0]}, "work must be"),
])
def test_attention_that_is_refused(native, q, pos, kw, match):
    with pytest.raises(ValueError, match=match):
        paged_decode_attention_fp8(q, *_cache(), TABLE, pos, **{"scale": 0.1, **kw})


U = torch.zeros(4)


@pytest.mark.parametrize("z,u,kw,match", [
    (_z(4), U, {}, "takes bf16 or fp32 logits"),
    (_z(4, 9, dtype=torch.float16), U, {}, "takes bf16 or fp32 logits"),
    (_z(4, 0), U, {}, "1 to 2\\^20"),
    (torch.zeros(1, 1).expand(4, (1 << 20) + 1), U, {}, "1 to 2\\^20"),
    (_z(4, 9), U[:3], {}, "uniforms must be"),
    (_z(4, 9), U.double(), {}, "uniforms must be"),
    (_z(4, 9), U, {"temperature": U[:2]}, "temperature must be"),
    (_z(4, 9), U, {"temperature": U.long()}, "temperature must be"),
    (_z(4, 9), U, {"top_k": U}, "top_k must be"),
    (_z(4, 9), U, {"top_k": U.bool()}, "top_k must be"),
    (_z(4, 9), U, {"top_p": U[:, None]}, "top_p must be"),
    (_z(4, 9), U, {"min_p": U.int()}, "min_p must be"),
])
def test_draws_that_are_refused(native, z, u, kw, match):
    with pytest.raises(ValueError, match=match):
        sample_tokens(z, u, **kw)


INVALID, UNSUPPORTED = 1, 2


def test_c_entries_check_before_a_launch():
    lib, n, at = _lib.lib(), None, 4096  # (an aligned address that is never read)

    def cache(k=at, v=at, ks=at, kps=4096, khs=2048, vps=4096, ksp=2, ksh=1, pages=8, table=at, cols=4):
        return (k, kps, khs, v, vps, 2048, ks, ksp, ksh, at, 2, 1, pages, table, cols, cols)

    def write(B=2, n_=3, heads=2, hd=128, q=at, st=256, lens=n, pos=at, **kw):
        return lib.evo2_kv_fp8_write(q, 3 * st, st, 128, at, 3 * st, st, 128, *cache(**kw), pos, lens, B, n_, heads, hd, n)

    def read(B=2, L=5, hd=128, out=at, lens=at, **kw):
        return lib.evo2_kv_fp8_read(*cache(**kw), lens, out, at, B, L, 2, hd, n)

    def rotary(B=2, hd=128, qkv=at, **kw):
        return lib.evo2_rotary_decode_fp8(qkv, 768, at, 1.0, at, *cache(**kw), at, B, 2, hd, n)

    need = lib.evo2_decode_attention_fp8_workspace_bytes(2, 1, 8, 2, 128, 400, 0)

    def attend(B=2, n_=1, heads=8, kv=2, hd=128, scale=0.1, q=at, qh=128, ws=at, bytes=need, shared=0, cols=400, **kw):
        return lib.evo2_paged_decode_attention_fp8(q, 1024, 1024, qh, *cache(cols=cols, **kw), shared, at, ws, bytes, at,
                                                   1024, 1024, 128, B, n_, heads, kv, hd, scale, n)

    for call in (write, read, rotary, attend):
        assert call(B=0) == 0
        assert call(B=-1) == INVALID
        assert call(hd=96) == UNSUPPORTED
        assert call(k=n) == INVALID and call(ks=n) == INVALID and call(table=n) == INVALID
        assert call(pages=0) == INVALID and call(cols=0) == INVALID and call(cols=(1 << 26) + 1) == INVALID
        assert call(k=at + 8) == UNSUPPORTED and call(khs=2040) == UNSUPPORTED
        assert call(khs=1024) == UNSUPPORTED and call(vps=4104) == UNSUPPORTED
    for call in (write, rotary):  # pages and scales that lie over one another are not written
        assert call(kps=0) == UNSUPPORTED and call(kps=2048) == UNSUPPORTED and call(kps=4080) == UNSUPPORTED
        assert call(vps=0) == UNSUPPORTED and call(ksp=0) == UNSUPPORTED and call(ksp=1) == UNSUPPORTED
        assert call(ksh=0) == UNSUPPORTED and b"overlap" in lib.evo2_last_error()
        assert call(kps=4096, khs=4096) == UNSUPPORTED and call(kps=2048, khs=7 * 2048) == UNSUPPORTED
    assert write(n_=0) == 0 and write(n_=-1) == INVALID and write(n_=1 << 31) == INVALID
    assert write(q=n) == INVALID and write(pos=n) == INVALID and write(q=at + 8) == UNSUPPORTED
    assert write(st=252) == UNSUPPORTED and write(B=65536) == UNSUPPORTED and write(heads=0) == INVALID
    assert read(L=0) == 0 and read(L=-1) == INVALID and read(lens=n) == INVALID and read(out=at + 2) == UNSUPPORTED
    assert rotary(qkv=n) == INVALID and rotary(B=65536) == UNSUPPORTED
    assert need > 0
    assert attend(n_=0) == 0 and attend(heads=7) == INVALID and attend(kv=0) == INVALID
    assert attend(scale=0.0) == INVALID and attend(scale=float("nan")) == INVALID
    assert attend(shared=401) == INVALID and attend(shared=-1) == INVALID
    assert attend(q=n) == INVALID and attend(q=at + 8) == UNSUPPORTED and attend(qh=132) == UNSUPPORTED
    assert attend(bytes=need - 1) == INVALID and attend(ws=n) == INVALID and b"workspace" in lib.evo2_last_error()
    assert attend(B=300, n_=300, bytes=1 << 62) == UNSUPPORTED and b"workgroups" in lib.evo2_last_error()

    def sample(B=2, V=9, z=at, sz=16, ws=at, bytes=1 << 40, u=at):
        return lib.evo2_sample(z, 1, sz, u, n, 1.0, n, 0, n, 1.0, n, 0.0, ws, bytes, at, B, V, n)

    assert sample(B=0) == 0 and sample(B=-1) == INVALID and sample(V=0) == INVALID
    assert sample(V=(1 << 20) + 1, sz=1 << 21) == INVALID
    assert sample(z=n) == INVALID and sample(u=n) == INVALID and sample(sz=8) == UNSUPPORTED
    assert sample(V=9000, sz=9000, bytes=64) == INVALID and sample(V=9000, sz=9000, ws=n) == INVALID
    assert sample(V=9000, sz=9000, ws=at + 8) == INVALID and b"workspace" in lib.evo2_last_error()
    assert sample(V=9000, sz=9000, B=65536) == UNSUPPORTED and b"workgroups" in lib.evo2_last_error()


def test_workspaces():
    lib = _lib.lib()
    need = lib.evo2_decode_attention_fp8_workspace_bytes
    for B, n, heads, kv, hd, pages, shared in ((1, 1, 32, 32, 128, 49, 0), (64, 1, 32, 32, 128, 545, 0), (8, 4, 32, 4, 64, 4096, 0),
                                               (32, 1, 64, 64, 128, 8195, 8192), (2, 1, 2, 1, 64, 1 << 22, 0),
                                               (65535, 1, 1, 1, 64, 1, 0)):
        rows = B * n * heads
        bytes = need(B, n, heads, kv, hd, pages, shared)
        # parts of at least 64 positions
        assert 0 <= bytes <= rows * (-(-pages * 16 // 64) + 1) * (hd + 2) * 4
        assert bytes % (rows * (hd + 2) * 4) == 0
    assert need(4, 1, 4, 4, 128, 4, 0) == 0  # one chunk: written out at once
    # a workgroup to a sequence: short, or as many as CUs; not of long ones, or behind shared pages
    assert need(64, 1, 4, 4, 128, 44, 0) == 0 and need(37, 1, 7, 7, 64, 44, 0) > 0 == need(2, 1, 128, 128, 128, 44, 0) == 0
    assert need(8, 1, 32, 32, 128, 1024, 0) == 0 < need(8, 1, 32, 32, 128, 1025, 0)
    assert need(1, 1, 32, 32, 128, 128, 0) > 0 and need(4, 1, 4, 4, 128, 60, 20) > 0
    assert need(0, 1, 4, 4, 128, 4, 0) == 0 and need(4, 1, 4, 3, 128, 4, 0) == 0 and need(4, 1, 4, 4, 128, 4, 5) == 0
    for B, V in ((64, 1024), (70000, 4096), (256, 8192)):  # a wave or a workgroup to a row
        assert lib.evo2_sample_workspace_bytes(B, V) == 0
    assert lib.evo2_sample_workspace_bytes(257, 8192) > 0 < lib.evo2_sample_workspace_bytes(1, 8193)
    ws = lib.evo2_sample_workspace_bytes(64, 131072)
    assert 64 * 131072 * 4 <= ws <= 64 * 131072 * 6
    assert lib.evo2_sample_workspace_bytes(0, 131072) == 0 == lib.evo2_sample_workspace_bytes(4, (1 << 20) + 1)


def test_shapes_of_a_call_reach_the_kernel(monkeypatch):
    """Strides and sizes as the C entry gets them: tokens of a projection's rows stay a view."""
    calls = []
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t=None: None)
    monkeypatch.setattr(_lib, "on_device", lambda t: _lib._HERE)
    monkeypatch.setattr(_lib, "call", lambda name, *a: calls.append((name, a)))
    c = _cache(hd=128)
    rows = _z(3, 7, 3 * 2 * 128)
    v = rows[..., 512:].view(3, 7, 2, 128)
    k = _z(3, 7, 2, 128)
    write_kv_fp8(k, v, *c, TABLE, POS.int(), POS)
    name, a = calls.pop()
    assert name == "evo2_kv_fp8_write" and len(a) == len(_lib.SIGNATURES[name])
    assert a[:4] == (k.data_ptr(), 7 * 256, 256, 128) and a[4:8] == (v.data_ptr(), 7 * 768, 768, 128)
    assert a[-5:-1] == (3, 7, 2, 128) and a[-6] == POS.data_ptr()
    q = _z(3, 5, 4, 128)[:, 1:3]
    out = paged_decode_attention_fp8(q, *c, TABLE, POS, 0.5, shared_pages=2)
    name, a = calls.pop()
    assert name == "evo2_paged_decode_attention_fp8" and len(a) == len(_lib.SIGNATURES[name])
    assert out.shape == q.shape and a[:4] == (q.data_ptr(), 5 * 512, 512, 128) and a[-7:-2] == (3, 2, 4, 2, 128)
    read_kv_fp8(*c, TABLE, POS, 33)
    name, a = calls.pop()
    assert len(a) == len(_lib.SIGNATURES[name]) and a[-5:-1] == (3, 33, 2, 128)
    z = _z(4, 20)[:, 3:12]
    sample_tokens(z, U, top_k=torch.tensor([1, 2, 3, 1 << 40]))
    name, a = calls.pop()
    assert len(a) == len(_lib.SIGNATURES[name]) and a[0] == z.data_ptr() and a[2] == 20
    assert a[5] == 1.0 and a[6] and a[-3:-1] == (4, 9)
    for k, want in ((1 << 70, 2 ** 31 - 1), (-(1 << 70), 0), (True, 1)):
        sample_tokens(z, U, top_k=k)
        assert calls.pop()[1][7] == want
    with pytest.raises(TypeError):
        sample_tokens(z, U, top_k=2.5)


def test_models_take_two_page_types():
    from evo2_flash_amd.config import HyenaConfig
    from evo2_flash_amd.model import Evo2Attention
    cfg = HyenaConfig(hidden_size=256, num_hidden_layers=1, num_attention_heads=4, intermediate_size=384, vocab_size=512,
                      hcs_layer_idxs=[], hcm_layer_idxs=[], hcl_layer_idxs=[], attn_layer_idxs=[0])
    a = Evo2Attention(cfg, 9, 4, 2, device="cpu", kv_dtype=F8)
    assert isinstance(a.cache, Fp8KVCache) and a.cache.k.dtype == F8
    with pytest.raises(ValueError, match="kv_dtype"):
        Evo2Attention(cfg, 9, 4, 2, device="cpu", kv_dtype=torch.int8)
