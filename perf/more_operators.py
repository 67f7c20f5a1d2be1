"""Cases of the operators of a decode loop over an 8-bit cache: writing the cache and reading
it back (`kv_fp8.write_kv_fp8`, `kv_fp8.read_kv_fp8`), decode attention over it
(`kv_fp8.paged_decode_attention_fp8`) and drawing the next token from the logits
(`sampling.sample_tokens`).

`run` makes one pass on what `prepare` gives: with `own` through the package's entry points,
else in elementary torch operations.  `exact` computes the same in 64 bits from the
definitions.

The cache: pages of 16 positions named by a block table, e4m3 codes with one power of two a
(page, head) as their scale, keys (pages, heads, 16, head_dim), values (pages, heads,
head_dim, 16).  The scale is the smallest with which no value of the page's tokens is over
448; a page that gets tokens behind ones it holds never lowers it, and re-encodes those where
it rises.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn
PAGE = 16
EMIN, EMAX = -110, 119


def listed():
    return [
        # one decode step's tokens of eight sequences, behind what their pages hold: latency
        {"name": "cache_step", "op": "cache", "starts": "1,15,16,31,33,46,47,62", "lens": "", "n": 1,
         "kv": 32, "hd": 128},
        # ragged reads of one padded batch, some of them further pieces of what was written
        # before, with shared key heads and heads of 64
        {"name": "cache_ragged", "op": "cache", "starts": "0,0,5,0,16,0,77,0,0,130,0,3",
         "lens": "700,1,333,1024,65,129,511,64,0,800,255,31", "n": 1024, "kv": 4, "hd": 64},
        # the 7B shape's prompt of 32768 tokens
        {"name": "cache_prompt_32k", "op": "cache", "starts": "0", "lens": "", "n": 32768, "kv": 32,
         "hd": 128},
        # one sequence of the 7B shape early in its answer: latency
        {"name": "attend_one", "op": "attend", "lens": "777", "n": 1, "heads": 32, "kv": 32,
         "hd": 128, "shared": 0},
        # the 7B shape at decode batch 8
        {"name": "attend_8x8k", "op": "attend",
         "lens": "8192,8193,8300,8447,8448,8600,8703,8704", "n": 1, "heads": 32, "kv": 32, "hd": 128,
         "shared": 0},
        # four draft tokens a request to verify, eight query heads to a key head, heads of 64
        {"name": "attend_verify", "op": "attend",
         "lens": "1,17,300,999,1024,1500,2047,2048,2500,3001,64,5,3500,3999,4000,16", "n": 4,
         "heads": 32, "kv": 4, "hd": 64, "shared": 0},
        # the 7B shape at decode batch 64, context 8192 and up
        {"name": "attend_64x8k", "op": "attend", "lens": ",".join(str(8192 + 8 * i) for i in range(64)),
         "n": 1, "heads": 32, "kv": 32, "hd": 128, "shared": 0},
        # the 40B shape: 32 sequences behind one prompt of 131072 tokens
        {"name": "attend_shared_131k", "op": "attend",
         "lens": ",".join(str(131073 + i) for i in range(32)), "n": 1, "heads": 64, "kv": 64,
         "hd": 128, "shared": 131072},
        # nucleotides: eight sequences' next tokens among the four likeliest
        {"name": "sample_8x512", "op": "sample", "rows": 8, "vocab": 512, "dtype": "bf16", "t": 1.0,
         "k": 4, "p": 1.0, "m": 0.0, "by_row": False},
        # many sequences, each with settings of its own, an odd vocabulary
        {"name": "sample_777x509", "op": "sample", "rows": 777, "vocab": 509, "dtype": "fp32", "t": 0.7,
         "k": 40, "p": 0.9, "m": 0.05, "by_row": True},
        # one sequence with a large vocabulary
        {"name": "sample_1x131072", "op": "sample", "rows": 1, "vocab": 131072, "dtype": "fp32",
         "t": 0.8, "k": 0, "p": 0.95, "m": 0.0, "by_row": False},
        # a decode batch of 64 with a large vocabulary, settings by row
        {"name": "sample_64x131072", "op": "sample", "rows": 64, "vocab": 131072, "dtype": "bf16",
         "t": 0.9, "k": 200, "p": 0.95, "m": 0.02, "by_row": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "sample"])
    hd = rng.choice([64, 128])
    if op == "cache":
        B, n, kv = _spread(rng, 1, 32), _spread(rng, 1, 4096), rng.choice([1, 2, 4, 8, 32])
        lens = "" if rng.random() < 0.4 else ",".join(str(rng.randint(0, n)) for _ in range(B))
        return {"op": op, "starts": ",".join(str(rng.choice([0, _spread(rng, 1, 300)])) for _ in range(B)),
                "lens": lens, "n": n, "kv": kv, "hd": hd}
    if op == "attend":
        B, kv = _spread(rng, 1, 48), rng.choice([1, 2, 4, 8, 32])
        shared = rng.choice([0, 0, 16 * _spread(rng, 1, 600)])
        top = max(2, min(16000, (1 << 23) // (B * kv)))
        return {"op": op, "lens": ",".join(str(shared + _spread(rng, 1, top)) for _ in range(B)),
                "n": rng.choice([1, 1, 1, 2, 5]), "heads": kv * rng.choice([1, 2, 4, 8]), "kv": kv,
                "hd": hd, "shared": shared}
    rows = _spread(rng, 1, 1500)
    return {"op": op, "rows": rows, "vocab": _spread(rng, 2, min(262144, (1 << 23) // rows)),
            "dtype": rng.choice(["bf16", "fp32"]), "t": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
            "k": rng.choice([0, 1, 4, 50, 1000]), "p": rng.choice([1.0, 0.95, 0.5]),
            "m": rng.choice([0.0, 0.02, 0.3]), "by_row": rng.random() < 0.5}


def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


def _take(pages, page):
    """pages[page] in 32 bits (8-bit floats are indexed as bytes)."""
    return pages.view(torch.uint8)[page].view(F8).float()


def _random_pages(pages, kv, hd, g):
    """Pages of e4m3 codes and their scales as a cache holds them: values of a few sizes, the
    largest of each (page, head) using the codes' top binade (keys; values by head and dim)."""
    codes = torch.empty(pages, kv, PAGE, hd, dtype=F8, device=DEV)
    scale = torch.empty(pages, kv, device=DEV)
    step = max(1, (1 << 26) // (kv * PAGE * hd))
    for at in range(0, pages, step):
        m = min(step, pages - at)
        x = torch.randn(m, kv, PAGE, hd, generator=g, device=DEV)
        x *= torch.exp2(torch.rand(m, kv, 1, 1, generator=g, device=DEV) * 2 - 0.8)
        e = _exponent(x.abs().amax((2, 3)))
        codes[at:at + m] = torch.ldexp(x, -e[:, :, None, None]).to(F8)
        scale[at:at + m] = torch.ldexp(torch.ones_like(x[:, :, 0, 0]), e)
    return codes, scale


def _exponent(amax):
    """The smallest e in [EMIN, EMAX] with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    frac, e = torch.frexp(amax)  # amax = frac * 2^e, frac in [0.5, 1)
    e = e - 9 + (frac > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, EMIN).clamp(EMIN, EMAX)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "sample":
        B, V = case["rows"], case["vocab"]
        dtype = BF if case["dtype"] == "bf16" else torch.float32
        z = torch.randn(B, V, generator=g, device=DEV) * 2.5
        if V >= 128:  # a few likely tokens, as a trained head gives
            z[:, torch.randint(V, (8,), generator=g, device=DEV)] += 6.0
        z[:, V - V // 100:] = float("-inf")  # a padded vocabulary's tail
        s.update(logits=z.to(dtype), u=torch.rand(B, generator=g, device=DEV))
        if case["by_row"]:
            jitter = torch.rand(B, generator=g, device=DEV)
            s.update(t=case["t"] * (0.5 + jitter), p=(case["p"] + 0.05 * (jitter - 1)),
                     k=torch.where(jitter < 0.2, 0, case["k"]).to(torch.int32), m=case["m"] * jitter)
        return s
    kv, hd, n = case["kv"], case["hd"], case["n"]
    if case["op"] == "cache":
        starts = _ints(case["starts"])
        lens = _ints(case["lens"]) or [n] * len(starts)
        need = [-(-(a + n) // PAGE) for a in starts]
        pages, B = sum(need) + 1, len(starts)
        table = torch.full((B, max(need)), -1, dtype=torch.int32, device=DEV)
        perm = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).to(torch.int32)
        ends = np.cumsum([0] + need)
        for b in range(B):
            table[b, :need[b]] = perm[ends[b]:ends[b + 1]]
        # the step's rows (q | k | v) of the projection: k as the rotary leaves it, v a view
        rows = torch.randn(B, n, 2 * kv, hd, generator=g, device=DEV).to(BF)
        rows *= torch.exp2(torch.rand(B, n, 2 * kv, 1, generator=g, device=DEV) * 3 - 1.5).to(BF)
        s.update(k=rows[:, :, :kv].contiguous(), v=rows[:, :, kv:], table=table,
                 positions=torch.tensor(starts, device=DEV),
                 lengths=torch.tensor(lens, device=DEV) if case["lens"] else None,
                 ends=torch.tensor([a + m for a, m in zip(starts, lens)], device=DEV),
                 L=max(a + m for a, m in zip(starts, lens)))
    else:
        lens, sp = _ints(case["lens"]), case["shared"] // PAGE
        B = len(lens)
        need = [-(-(m + n - 1) // PAGE) - sp for m in lens]
        pages = sp + sum(need) + 1
        table = torch.full((B, sp + max(need)), -1, dtype=torch.int32, device=DEV)
        perm = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).to(torch.int32)
        table[:, :sp] = perm[:sp]
        ends = np.cumsum([sp] + need)
        for b in range(B):
            table[b, sp:sp + need[b]] = perm[ends[b]:ends[b + 1]]
        heads = case["heads"]
        q = (torch.randn(B, n, heads, hd, generator=g, device=DEV) * 1.28).to(BF)
        s.update(q=q[:, 0] if n == 1 else q, table=table,
                 positions=torch.tensor([m - 1 for m in lens], device=DEV), scale=hd ** -0.5)
    s["kp"], s["ks"] = _random_pages(pages, kv, hd, g)
    vp, s["vs"] = _random_pages(pages, kv, hd, g)
    s["vp"] = vp.view(pages, kv, hd, PAGE)
    return s


# ------------------------------------------------------------ plain forms

def _plain_write(x, pages, scale, s, turned):
    """x (B, n, kv, hd) into pages (P, kv, 16, hd) (turned: (P, kv, hd, 16)), in place."""
    B, n, kv, hd = x.shape
    start = s["positions"]
    count = torch.full_like(start, n) if s["lengths"] is None else s["lengths"]
    cols = torch.arange(-(-n // PAGE) + 1, device=x.device)
    col = start[:, None] // PAGE + cols                                  # (B, C) table columns
    pos = col[:, :, None] * PAGE + torch.arange(PAGE, device=x.device)   # (B, C, 16)
    token = pos - start[:, None, None]
    new = (token >= 0) & (token < count[:, None, None])
    col = col.clamp(max=s["table"].shape[1] - 1)
    b, c = torch.nonzero(new.any(2), as_tuple=True)                      # the pages written
    page = s["table"][b, col[b, c]].long()
    token, new = token[b, c], new[b, c][:, None, :, None]                # (W, 16), (W, 1, 16, 1)
    old = (token < 0)[:, None, :, None]
    xs = x[b[:, None], token.clamp(0, n - 1)].float().transpose(1, 2)     # (W, kv, 16, hd)
    e = _exponent(torch.where(new, xs, 0.0).abs().amax((2, 3)))
    held = torch.frexp(scale[page])[1] - 1
    e = torch.where(old.any(2)[:, :, 0], torch.maximum(e, held), e)
    was = _take(pages, page).transpose(2, 3) if turned else _take(pages, page)
    values = torch.ldexp(was, (held - e)[:, :, None, None])
    values = torch.where(new, torch.ldexp(xs, -e[:, :, None, None]).clamp(-448, 448), values)
    codes = torch.where(new | old, values, was).to(F8).view(torch.uint8)
    pages.view(torch.uint8)[page] = codes.transpose(2, 3) if turned else codes
    scale[page] = torch.ldexp(torch.ones_like(scale[page]), e)


def _plain_read(pages, scale, s, turned):
    cols = -(-s["L"] // PAGE)
    page = s["table"][:, :cols].long().clamp(min=0)
    x = _take(pages, page) * scale[page][..., None, None]               # (B, C, kv, ., .)
    x = x.permute(0, 1, 4, 2, 3) if turned else x.transpose(2, 3)        # (B, C, 16, kv, hd)
    x = x.flatten(1, 2)[:, :s["L"]]
    live = torch.arange(s["L"], device=x.device) < s["ends"][:, None]
    return torch.where(live[..., None, None], x, 0.0).to(BF)


def _plain_cache(s):
    _plain_write(s["k"], s["kp"], s["ks"], s, False)
    _plain_write(s["v"], s["vp"], s["vs"], s, True)
    return {"k": _plain_read(s["kp"], s["ks"], s, False), "v": _plain_read(s["vp"], s["vs"], s, True),
            "k_scale": s["ks"], "v_scale": s["vs"]}


def _plain_dense(s, table):
    """The keys and values (B, kv, positions, hd) of a table's pages in 32 bits."""
    page = table.long().clamp(min=0)
    k = _take(s["kp"], page) * s["ks"][page][..., None, None]           # (B, C, kv, 16, hd)
    v = _take(s["vp"], page) * s["vs"][page][..., None, None]           # (B, C, kv, hd, 16)
    return k.transpose(1, 2).flatten(2, 3), v.permute(0, 2, 1, 4, 3).flatten(2, 3)


def _plain_attend(s):
    B, n, heads, kv, hd = len(s["positions"]), s["n"], s["heads"], s["kv"], s["hd"]
    q = s["q"].float().view(B, n, kv, heads // kv, hd).permute(2, 0, 1, 3, 4)
    q = q.reshape(kv, B, n * (heads // kv), hd)                          # (kv, B, rows, hd)
    rows, sp = q.shape[2], s["shared"] // PAGE
    # the shared pages once for all sequences, then each sequence's own
    k0, v0 = _plain_dense(s, s["table"][:1, :sp])
    k1, v1 = _plain_dense(s, s["table"][:, sp:])
    s0 = torch.matmul(q.reshape(kv, B * rows, hd), k0[0].transpose(1, 2)).view(kv, B, rows, sp * PAGE)
    s1 = torch.matmul(q, k1.permute(1, 0, 3, 2))
    sc = torch.cat([s0, s1], -1) * s["scale"]
    last = s["positions"][:, None] + torch.arange(n, device=q.device)    # (B, n)
    last = last.repeat_interleave(heads // kv, 1)
    live = torch.arange(sc.shape[-1], device=q.device) <= last[..., None]
    sc = sc.masked_fill(~live, float("-inf"))
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    p0, p1 = p[..., :sp * PAGE], p[..., sp * PAGE:]
    out = torch.matmul(p1, v1.transpose(0, 1))
    out = out + torch.matmul(p0.reshape(kv, B * rows, sp * PAGE), v0[0]).view(out.shape)
    out = out.view(kv, B, n, heads // kv, hd).permute(1, 2, 0, 3, 4).reshape(B, n, heads, hd)
    return {"out": (out[:, 0] if n == 1 else out).to(BF)}


def _settings(s):
    """Temperature, k, p and the least share by row, the numbers held as in 32 bits."""
    B, dev = s["logits"].shape[0], s["logits"].device
    give = lambda x, dtype: torch.as_tensor(x, dtype=dtype, device=dev).expand(B)[:, None]  # noqa: E731
    return (give(s["t"], torch.float32).double(), give(s["k"], torch.int64),
            give(s["p"], torch.float32).double(), give(s["m"], torch.float32).double())


def _plain_sample(s):
    # in 64 bits: the running sums decide between neighbouring tokens
    z, u = s["logits"].double(), s["u"].double()[:, None]
    t, k, p, m = _settings(s)
    z, order = torch.sort(z, dim=1, descending=True, stable=True)          # ties: lowest index first
    w = torch.exp((z - z[:, :1]) / torch.where(t > 0, t, 1.0))
    at = torch.arange(z.shape[1], device=z.device)
    keep = (at < torch.where(k > 0, k, z.shape[1])) & (z > float("-inf"))
    w = torch.where(keep, w, 0.0)
    before = w.cumsum(1) - w
    keep &= (before < p * w.sum(1, keepdim=True)) | (p >= 1)
    keep &= w >= m
    keep &= (t > 0) | (at == 0)
    keep[:, 0] = True
    # back in the vocabulary's order: the first token whose running sum passes u * total
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run = w.cumsum(1)
    return {"token": (run <= u * run[:, -1:]).sum(1)}


# ------------------------------------------------------------ the package's calls

def _own_cache(s):
    from evo2_flash_amd.kv_fp8 import read_kv_fp8, write_kv_fp8
    cache = (s["kp"], s["vp"], s["ks"], s["vs"])
    write_kv_fp8(s["k"], s["v"], *cache, s["table"], s["positions"], s["lengths"])
    k, v = read_kv_fp8(*cache, s["table"], s["ends"], s["L"])
    return {"k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}


def _own_attend(s):
    from evo2_flash_amd.kv_fp8 import paged_decode_attention_fp8
    return {"out": paged_decode_attention_fp8(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"],
                                              s["positions"], s["scale"],
                                              shared_pages=s["shared"] // PAGE)}


def _own_sample(s):
    from evo2_flash_amd.sampling import sample_tokens
    return {"token": sample_tokens(s["logits"], s["u"], temperature=s["t"], top_k=s["k"],
                                   top_p=s["p"], min_p=s["m"])}


def run(state):
    if not own:
        return {"cache": _plain_cache, "attend": _plain_attend, "sample": _plain_sample}[state["op"]](state)
    return {"cache": _own_cache, "attend": _own_attend, "sample": _own_sample}[state["op"]](state)


# ------------------------------------------------------------ work and 64 bits

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 12 * case["rows"], "flops": 4 * n}
    kv, hd, n = case["kv"], case["hd"], case["n"]
    if case["op"] == "cache":
        starts = _ints(case["starts"])
        lens = _ints(case["lens"]) or [n] * len(starts)
        L = max(a + m for a, m in zip(starts, lens))
        written = sum(lens)
        pages = sum(-(-(a + m) // PAGE) for a, m in zip(starts, lens))
        read = sum(a + m for a, m in zip(starts, lens))
        # k and v: tokens in as bf16, codes out; codes in, bf16 out with the zeros behind
        return {"bytes": 2 * (kv * hd * (3 * written + read + 2 * len(starts) * L) + 8 * kv * pages),
                "flops": 2 * 2 * kv * hd * (written + read)}
    lens, heads, shared = _ints(case["lens"]), case["heads"], case["shared"]
    held = shared + sum(m + n - 1 - shared for m in lens)  # positions read, shared ones once
    pairs = sum(n * m + n * (n - 1) // 2 for m in lens)
    return {"bytes": 2 * kv * (held * hd + 4 * -(-held // PAGE)) + 2 * 2 * len(lens) * n * heads * hd,
            "flops": 4 * heads * hd * pairs}


def _round_e4m3(y):
    """y in 64 bits to the nearest e4m3 value, ties to even, saturated at 448."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # of y's binade
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_side(x, codes, scale, table, starts, lens, L):
    """Write x's tokens page by page and read L positions back in 64 bits: codes
    (P, 16, kv, hd) and scale (P, kv), both changed in place."""
    out = x.new_zeros(len(starts), L, x.shape[2], x.shape[3])
    binades = torch.exp2(torch.arange(EMIN, EMAX + 1, device=x.device, dtype=torch.float64))
    for b, (a, m) in enumerate(zip(starts, lens)):
        for c in range(a // PAGE, -(-(a + m) // PAGE) if m else 0):
            pg, lo, hi = table[b][c], max(a - c * PAGE, 0), min(a + m - c * PAGE, PAGE)
            t = x[b, c * PAGE + lo - a:c * PAGE + hi - a]                # (tokens, kv, hd)
            # the first power of two that 448 of reach the largest value
            now = binades[torch.searchsorted(448 * binades, t.abs().amax((0, 2))).clamp(max=EMAX - EMIN)]
            if lo:
                now = torch.maximum(now, scale[pg])
                codes[pg, :lo] = _round_e4m3(codes[pg, :lo] * (scale[pg] / now)[:, None])
            codes[pg, lo:hi] = _round_e4m3(t / now[:, None])
            scale[pg] = now
        for c in range(-(-(a + m) // PAGE)):
            pg, hi = table[b][c], min(a + m - c * PAGE, PAGE)
            out[b, c * PAGE:c * PAGE + hi] = codes[pg, :hi] * scale[pg][:, None]
    return out, scale


def _exact_cache(case, s):
    starts = _ints(case["starts"])
    lens = _ints(case["lens"]) or [case["n"]] * len(starts)
    table = s["table"].tolist()
    k, ks = _exact_side(s["k"].double(), s["kp"].double().transpose(1, 2).contiguous(), s["ks"].double(),
                        table, starts, lens, s["L"])
    v, vs = _exact_side(s["v"].double(), s["vp"].double().permute(0, 3, 1, 2).contiguous(), s["vs"].double(),
                        table, starts, lens, s["L"])
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _exact_attend(case, s):
    n, group = case["n"], case["heads"] // case["kv"]
    lens, sp = _ints(case["lens"]), case["shared"] // PAGE
    B, hd = len(lens), case["hd"]
    q = s["q"].double().view(B, n, case["heads"], hd)
    out = torch.zeros_like(q)

    def values(pages, j):  # key head j of some pages: (positions, hd) each
        k = _take(s["kp"][:, j], pages).double() * s["ks"][pages, j, None, None].double()
        v = _take(s["vp"][:, j], pages).double() * s["vs"][pages, j, None, None].double()
        return k.reshape(-1, hd), v.transpose(1, 2).reshape(-1, hd)

    for j in range(case["kv"]):
        h = slice(j * group, (j + 1) * group)
        front = values(s["table"][0, :sp].long(), j)
        for b, m in enumerate(lens):
            own_pages = s["table"][b, sp:-(-(m + n - 1) // PAGE)].long()
            k, v = (torch.cat(t) for t in zip(front, values(own_pages, j)))
            for i in range(n):
                p = torch.softmax((q[b, i, h] * s["scale"]) @ k[:m + i].t(), 1)
                out[b, i, h] = p @ v[:m + i]
    return {"out": out[:, 0] if n == 1 else out}


def _exact_sample(case, s):
    t, k, p, m = (x[:, 0].tolist() for x in _settings(s))
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().tolist()
    tokens = []
    for b, z in enumerate(logits):
        order = np.lexsort((np.arange(z.size), -z))
        order = order[np.isfinite(z[order])]
        if t[b] <= 0:
            tokens.append(int(order[0]))
            continue
        if k[b] > 0:
            order = order[:k[b]]
        w = np.exp((z[order] - z[order[0]]) / t[b])
        if p[b] < 1:
            run = np.cumsum(w)
            order = order[:1 + int((run[:-1] < p[b] * run[-1]).sum())]
        order = order[:max(1, int((w[:order.size] >= m[b]).sum()))]
        kept = np.sort(order)
        run = np.cumsum(np.exp((z[kept] - z.max()) / t[b]))
        tokens.append(int(kept[min(kept.size - 1, int((run <= u[b] * run[-1]).sum()))]))
    return {"token": torch.tensor(tokens)}


def exact(case, seed):
    if case["op"] == "attend" and len(_ints(case["lens"])) * case["kv"] * case["n"] > 4096:
        return None  # a product a (sequence, head, token): too many to wait for
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)
