"""The decoder's KV cache in 8 bits, and decode attention over it (model.py:104-153): half
the bytes of the bf16 pages, which is what decode attention over long contexts waits for.

Keys and values are e4m3 codes in pages of 16 positions named by a block table, as in
attention.PagedKVCache, in the layouts the kernels load as they lie (csrc/kv_fp8.h):

    k_pages (pages, kv_heads, 16, head_dim)    v_pages (pages, kv_heads, head_dim, 16)
    k_scale, v_scale (pages, kv_heads) fp32    value = code * scale

The scale of a (page, head) is the smallest power of two, of 2^-110 .. 2^119, with which no
finite value written since the page's first position was is over 448 codes.  A token's place
in its page decides: the write of a page's first position starts the page's scale, a write
behind positions that the page holds keeps it, or raises it and re-encodes those (exactly, but
for codes that reach the subnormal range).  No other write lowers a scale: a large token that
is written over (a draft that was rejected) leaves its page the coarser steps.  NaN and
infinities are held as NaN.  Codes are rounded to nearest even.  A page that two sequences
share is only read: two sequences of one call that write to it leave it undefined.

write_kv_fp8, read_kv_fp8 and paged_decode_attention_fp8 take the tensors; Fp8KVCache holds
them for one attention layer.  rotary_decode_fp8 is the decode step's rotary with the write.
"""

import torch

from . import _lib
from .attention import PAGE, _page_table, _rotary_rows

_F8 = torch.float8_e4m3fn
_NO_SCALE = 2.0 ** -110  # of a page of zeros
_INTS = (torch.int32, torch.int64)


# The checks below run for every call of a decode step, which waits for the host: each of a
# tensor's properties is asked for once (attention of one sequence 20 -> 17 us a call).
def _cache_args(what, k_pages, v_pages, k_scale, v_scale, block_table, B):
    """Checks of the cache's tensors and the table; the C entries' arguments from the key
    pages to the table's columns, and (kv_heads, head_dim, device index)."""
    dev = k_pages.get_device()
    same = (dev == v_pages.get_device() == k_scale.get_device() == v_scale.get_device()
            == block_table.get_device())
    if dev < 0 or not same:
        _lib.require_device(k_pages, v_pages, k_scale, v_scale, block_table)
        if not same:
            raise ValueError(f"{what}: the cache and its table are on different devices")
    shape = k_pages.shape
    if len(shape) != 4 or shape[2] != PAGE or k_pages.dtype != _F8 or v_pages.dtype != _F8:
        raise ValueError(f"{what} takes float8_e4m3fn pages (pages, kv_heads, {PAGE}, head_dim) and "
                         f"(pages, kv_heads, head_dim, {PAGE}), got {tuple(shape)} {k_pages.dtype}, "
                         f"{tuple(v_pages.shape)} {v_pages.dtype}")
    pages, kv, _, hd = shape
    if v_pages.shape != (pages, kv, hd, PAGE):
        raise ValueError(f"{what}: page shapes {tuple(shape)}, {tuple(v_pages.shape)} do not match")
    if hd != 128 and hd != 64:
        raise ValueError(f"{what} takes head_dim 64 or 128, got {hd}")
    if (k_scale.shape != (pages, kv) or v_scale.shape != (pages, kv) or k_scale.dtype != torch.float32
            or v_scale.dtype != torch.float32):
        raise ValueError(f"{what}: scales must be ({pages}, {kv}) fp32, got {tuple(k_scale.shape)} "
                         f"{k_scale.dtype}, {tuple(v_scale.shape)} {v_scale.dtype}")
    if pages == 0 or kv == 0:
        raise ValueError(f"{what}: a cache of no pages or heads")
    kps, khs, k2, k3 = k_pages.stride()
    vps, vhs, v2, v3 = v_pages.stride()
    if k2 != hd or k3 != 1 or v2 != PAGE or v3 != 1:
        raise ValueError(f"{what}: a page's head must be contiguous")
    table = block_table.shape
    if len(table) != 2 or table[0] < B or table[1] == 0 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be (>= {B}, max_pages) int32, got {tuple(table)} "
                         f"{block_table.dtype}")
    row, unit = block_table.stride()
    if unit != 1 and table[1] != 1:
        raise ValueError("block_table must have unit column stride")
    return (k_pages.data_ptr(), kps, khs, v_pages.data_ptr(), vps, vhs, k_scale.data_ptr(),
            *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride(), pages, block_table.data_ptr(), row,
            table[1]), kv, hd, dev


def _on(dev, what, *tensors):
    """Refuse tensors that are not on the cache's device `dev`."""
    for t in tensors:
        if t.get_device() != dev:
            _lib.require_device(t)
            raise ValueError(f"{what}: a tensor on {t.device}, the cache on cuda:{dev}")


def _per_sequence(t, B, name, dev):
    """t (B,) int32 or int64 on the cache's device, as contiguous int64."""
    if t.shape != (B,) or t.dtype not in _INTS:
        raise ValueError(f"{name} must be ({B},) int32 or int64, got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != dev:
        _on(dev, name, t)
    if t.dtype == torch.int64 and (B <= 1 or t.stride(0) == 1):
        return t
    return t.to(torch.int64).contiguous()


def _token_rows(t):
    """t (B, n, heads, hd) with rows as the kernels read them: unit last stride, 16-byte
    aligned; (itself or a copy, address, batch, token and head stride)."""
    b, n, h, unit = t.stride()
    at = t.data_ptr()
    if unit != 1 or (b | n | h) & 7 or at & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        b, n, h, _ = t.stride()
        at = t.data_ptr()
    return t, at, b, n, h


def write_kv_fp8(k, v, k_pages, v_pages, k_scale, v_scale, block_table, positions, lengths=None):
    """Quantise k and v (B, n, kv_heads, head_dim) bf16 (views of any strides) into the
    cache's pages: token i of sequence b goes to position positions[b] + i of
    `block_table`'s (>= B, max_pages) int32 row b.  lengths (B,): only a sequence's first
    lengths[b] tokens count (a padded batch).  positions and lengths are int32 or int64 on
    the cache's device; the host does not read them.  Tokens whose position lies outside the
    table, or whose entry lies outside the cache's pages, are not written; nor is any token of
    a sequence that starts there.  Codes of positions that are not written keep their bytes
    (of positions held before theirs: see the module's description).  Pages that lie over one
    another (an expanded tensor) are refused, and so are more than 65535 sequences."""
    shape, bf = k.shape, torch.bfloat16
    if len(shape) != 4 or v.shape != shape or k.dtype != bf or v.dtype != bf:
        raise ValueError(f"write_kv_fp8 takes bf16 k and v (B, n, kv_heads, head_dim), got "
                         f"{tuple(shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
    B, n, heads, width = shape
    cache, kv, hd, dev = _cache_args("write_kv_fp8", k_pages, v_pages, k_scale, v_scale, block_table, B)
    if heads != kv or width != hd:
        raise ValueError(f"write_kv_fp8: tokens of ({heads}, {width}), pages of ({kv}, {hd})")
    _on(dev, "write_kv_fp8", k, v)
    positions = _per_sequence(positions, B, "positions", dev)
    if lengths is not None:
        lengths = _per_sequence(lengths, B, "lengths", dev)
    if B == 0 or n == 0:
        return
    k, *krow = _token_rows(k)
    v, *vrow = _token_rows(v)
    with _lib.on_device(k_pages):
        _lib.call("evo2_kv_fp8_write", *krow, *vrow, *cache, positions.data_ptr(), _lib.ptr(lengths), B,
                  n, kv, hd, _lib.stream_of(k_pages))


def read_kv_fp8(k_pages, v_pages, k_scale, v_scale, block_table, lengths, L):
    """The first L positions of sequences 0 .. B - 1 (B: lengths' size) as bf16 keys and
    values (B, L, kv_heads, head_dim), the values the codes stand for exactly (the layout of
    write_kv_fp8's tokens and, flattened, of attention.packed_attention's).  Positions from
    lengths[b] on, and those whose entry lies outside the table or the cache's pages, are
    zeros.  More than 65535 sequences are refused."""
    B, L = lengths.shape[0] if lengths.dim() else -1, int(L)
    cache, kv, hd, dev = _cache_args("read_kv_fp8", k_pages, v_pages, k_scale, v_scale, block_table, B)
    lengths = _per_sequence(lengths, B, "lengths", dev)
    if L < 0:
        raise ValueError(f"read_kv_fp8 takes L >= 0, got {L}")
    k = torch.empty((B, L, kv, hd), dtype=torch.bfloat16, device=k_pages.device)
    v = torch.empty_like(k)
    if B and L:
        with _lib.on_device(k_pages):
            _lib.call("evo2_kv_fp8_read", *cache, lengths.data_ptr(), k.data_ptr(), v.data_ptr(), B, L,
                      kv, hd, _lib.stream_of(k_pages))
    return k, v


def workspace_fp8(B, heads, kv_heads, head_dim, max_pages, device, n=1, shared_pages=0):
    """A workspace for paged_decode_attention_fp8 on up to B sequences of up to n tokens over
    tables of max_pages columns (a table of fewer can need more), with and without the shared
    pages (allocate once, outside graph capture; calls that may run at once take one each)."""
    need = max((_lib.workspace_bytes("evo2_decode_attention_fp8_workspace_bytes", b, m, heads,
                                     kv_heads, head_dim, max_pages, s)
                for b in range(1, B + 1) for m in range(1, n + 1) for s in {0, int(shared_pages)}),
               default=0)
    return torch.empty(max(need, 16), dtype=torch.uint8, device=device)


def paged_decode_attention_fp8(q, k_pages, v_pages, k_scale, v_scale, block_table, positions, scale,
                               work=None, shared_pages=0):
    """Attention of q (B, heads, head_dim), or n tokens of each sequence (B, n, heads,
    head_dim), bf16, over the cache; heads a multiple of kv_heads (query head h reads key
    head h // (heads // kv_heads)).  positions (B,): token i of sequence b attends to
    positions 0 .. positions[b] + i of block_table's (>= B, max_pages) int32 row b (those
    past the table do not exist).  Returns bf16 of q's shape: the exact softmax over the
    values the codes stand for (fp32 scores and sums, the probabilities to ~16 bits).

    The kernel never reads through a table entry outside [0, pages): its positions are left
    out of the softmax (a token with none left gets zeros).  shared_pages: the first
    shared_pages entries of every row name the same pages (attention.shared_prefix_pages
    finds them on the host), which are then read once for 32 query rows of any sequences.
    Bytes of positions that a token does not attend to may be anything.  No gradients are
    recorded.  The context is split for the table's columns: a table far longer than the
    sequences is passed as its first columns (777 positions of 32 heads 10 us, in a table of
    131072 positions 31), with a workspace of that width.  B * n over 65535, scales of 2.3e38
    and above and a `work` that is too small are refused; scores past fp32 give NaN."""
    shape = q.shape
    if len(shape) == 3:
        (B, heads, width), n = shape, 1
    elif len(shape) == 4:
        B, n, heads, width = shape
    if not 3 <= len(shape) <= 4 or q.dtype != torch.bfloat16:
        raise ValueError(f"paged_decode_attention_fp8 takes bf16 q (B, [n,] heads, head_dim), got "
                         f"{tuple(shape)} {q.dtype}")
    cache, kv, hd, dev = _cache_args("paged_decode_attention_fp8", k_pages, v_pages, k_scale, v_scale,
                                     block_table, B)
    if width != hd or heads == 0 or heads % kv:
        raise ValueError(f"paged_decode_attention_fp8: q {tuple(shape)} does not match pages "
                         f"{tuple(k_pages.shape)}")
    _on(dev, "paged_decode_attention_fp8", q)
    positions = _per_sequence(positions, B, "positions", dev)
    scale, shared_pages, max_pages = float(scale), int(shared_pages), cache[-1]
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"paged_decode_attention_fp8 takes a positive scale, got {scale}")
    if not 0 <= shared_pages <= max_pages:
        raise ValueError(f"shared_pages {shared_pages} of a table of {max_pages} columns")
    if work is not None and (not work.is_contiguous() or work.get_device() != dev):
        raise ValueError("work must be a contiguous tensor on the cache's device")
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    if B == 0 or n == 0:
        return out
    if len(shape) == 3:
        b, h, unit = q.stride()
        at = q.data_ptr()
        if unit != 1 or (b | h) & 7 or at & 15:
            q = q.clone(memory_format=torch.contiguous_format)
            b, h, _ = q.stride()
            at = q.data_ptr()
        row = at, b, 0, h
    else:
        q, *row = _token_rows(q)
    with _lib.on_device(q):
        if work is None:
            bytes = _lib.workspace_bytes("evo2_decode_attention_fp8_workspace_bytes", B, n, heads, kv, hd,
                                         max_pages, shared_pages)
            if bytes:
                work = torch.empty(bytes, dtype=torch.uint8, device=q.device)
        else:
            bytes = work.numel() * work.element_size()
        _lib.call("evo2_paged_decode_attention_fp8", *row, *cache, shared_pages, positions.data_ptr(),
                  _lib.ptr(work), bytes, out.data_ptr(), n * heads * hd, heads * hd, hd, B, n, heads, kv, hd,
                  scale, _lib.stream_of(q))
    return out


class Fp8KVCache:
    """One attention layer's 8-bit KV pages and their scales, zeros at first; page 0 is never
    handed out."""

    def __init__(self, num_pages, heads, head_dim, device):
        self.k = torch.zeros(num_pages, heads, PAGE, head_dim, dtype=torch.uint8, device=device).view(_F8)
        self.v = torch.zeros(num_pages, heads, head_dim, PAGE, dtype=torch.uint8, device=device).view(_F8)
        self.k_scale = torch.full((num_pages, heads), _NO_SCALE, dtype=torch.float32, device=device)
        self.v_scale = torch.full((num_pages, heads), _NO_SCALE, dtype=torch.float32, device=device)

    @property
    def tensors(self):
        """The tensors as write_kv_fp8 and the other operators take them."""
        return self.k, self.v, self.k_scale, self.v_scale

    def clear(self):
        """Zeros in every page, as a new cache has."""
        for t in (self.k, self.v):
            t.view(torch.uint8).zero_()
        self.k_scale.fill_(_NO_SCALE)
        self.v_scale.fill_(_NO_SCALE)

    def fill(self, values):
        """Every page's 16 tokens: values(pages, 16, heads, head_dim) makes keys and values
        for some pages at a time."""
        pages, heads, _, hd = self.k.shape
        step = max(1, min(65535, (1 << 27) // (PAGE * heads * hd)))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            table = torch.arange(at, at + n, dtype=torch.int32, device=self.k.device).view(n, 1)
            k, v = (values(n, PAGE, heads, hd).to(torch.bfloat16) for _ in range(2))
            write_kv_fp8(k, v, *self.tensors, table, torch.zeros(n, dtype=torch.int64, device=k.device))

    def append(self, k, v, block_table, positions):
        """k, v (B, heads, head_dim): the entries of sequence b at positions[b]."""
        write_kv_fp8(k[:, None], v[:, None], *self.tensors, block_table, positions)

    def write_prompt(self, k, v, block_table):
        """k, v (B, heads, L, head_dim): positions 0..L-1 of sequences 0..B-1."""
        zero = torch.zeros(k.shape[0], dtype=torch.int64, device=k.device)
        write_kv_fp8(k.transpose(1, 2), v.transpose(1, 2), *self.tensors, block_table, zero)

    def dense(self, block_table, B, L):
        """The first L positions of sequences 0..B-1 as contiguous bf16 caches (keys
        (B, heads, head_dim, L), values (B, heads, L, head_dim))."""
        lengths = torch.full((B,), L, dtype=torch.int64, device=self.k.device)
        k, v = read_kv_fp8(*self.tensors, block_table, lengths, L)
        return k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()


def rotary_prefill_fp8(qkv, cache, block_table, inv_freq, factor, nseq, L):
    """attention.rotary_prefill on an Fp8KVCache: the same operands of prefill attention (of
    the values before they are quantised); k and v are quantised into `cache`'s pages by a
    launch of their own, which reads them again (32768 tokens of 32 heads of 128 516 us, with
    bf16 pages, written in the one launch, 489)."""
    _lib.require_device(qkv, cache.k, cache.v, inv_freq)
    nh, hd = cache.k.shape[1], cache.k.shape[3]
    qkv, inv_freq = _rotary_rows(qkv, nh, hd, inv_freq)
    if qkv.shape[0] != nseq * L:
        raise ValueError(f"qkv must have {nseq * L} rows, got {qkv.shape[0]}")
    block_table = _page_table(block_table, nseq, cache.k.shape[0], qkv.device)
    Lv = -(-L // 128) * 128
    q = torch.empty(nseq, nh, L, hd, dtype=qkv.dtype, device=qkv.device)
    k = torch.empty_like(q)
    vt = torch.empty(nseq, nh, hd, Lv, dtype=qkv.dtype, device=qkv.device)
    with _lib.on_device(qkv):
        _lib.call("evo2_rotary_prefill", _lib.ptr(qkv), qkv.stride(0), _lib.ptr(inv_freq), float(factor),
                  _lib.ptr(q), _lib.ptr(k), _lib.ptr(vt), Lv, None, 0, 0, 0, None, 0, 0, 0, 0,
                  _lib.ptr(block_table), block_table.stride(0), block_table.shape[1], nseq, nh, hd, L,
                  _lib.stream_of(qkv))
    v = qkv[:, 2 * nh * hd:].view(nseq, L, nh, hd)
    zero = torch.zeros(nseq, dtype=torch.int64, device=qkv.device)
    write_kv_fp8(k.transpose(1, 2), v, *cache.tensors, block_table, zero)
    return q, k, vt


def rotary_decode_fp8(qkv, cache, block_table, positions, inv_freq, factor):
    """attention.rotary_decode on an Fp8KVCache, in one launch: qkv (B, 3 * heads *
    head_dim) bf16 rows (q | k | v) at positions (B,); returns q (B, heads, head_dim)
    rotated; k and v are quantised into `cache`'s pages as write_kv_fp8 does."""
    _lib.require_device(qkv, cache.k, cache.v, block_table, positions, inv_freq)
    nh, hd = cache.k.shape[1], cache.k.shape[3]
    qkv, inv_freq = _rotary_rows(qkv, nh, hd, inv_freq)
    B = qkv.shape[0]
    table = _page_table(block_table, B, cache.k.shape[0], qkv.device)
    args, _, _, dev = _cache_args("rotary_decode_fp8", *cache.tensors, table, B)
    _on(dev, "rotary_decode_fp8", qkv, inv_freq)
    positions = _per_sequence(positions, B, "positions", dev)
    q = torch.empty(B, nh, hd, dtype=qkv.dtype, device=qkv.device)
    with _lib.on_device(qkv):
        _lib.call("evo2_rotary_decode_fp8", _lib.ptr(qkv), qkv.stride(0), _lib.ptr(inv_freq), float(factor),
                  _lib.ptr(q), *args, _lib.ptr(positions), B, nh, hd, _lib.stream_of(qkv))
    return q


__all__ = ["Fp8KVCache", "write_kv_fp8", "read_kv_fp8", "paged_decode_attention_fp8", "workspace_fp8",
           "rotary_prefill_fp8", "rotary_decode_fp8"]
