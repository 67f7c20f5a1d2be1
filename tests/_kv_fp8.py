"""Plain 64-bit forms of the 8-bit KV cache on the host, for its tests: e4m3 codes with one
power of two a (page, head)."""

import torch

PAGE = 16
F8 = torch.float8_e4m3fn


def exponent(amax):
    """The smallest e of [-110, 119] with amax <= 448 * 2^e (amax: 64-bit values)."""
    e = torch.full(amax.shape, -110.0, dtype=torch.float64)
    for x in range(-110, 119):
        e = torch.where(amax > 448.0 * 2.0 ** x, x + 1.0, e)
    return e


def round_e4m3(y):
    """64-bit y to the nearest e4m3 value, ties to even, saturated; NaN and infinities NaN."""
    fine = torch.isfinite(y)
    a = torch.where(fine, y, 0.0)
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(fine, (torch.round(a / step) * step).clamp(-448, 448), float("nan"))


def write_side(x, pages, scale, table, positions, lengths):
    """x (B, n, kv, hd) into pages (P, kv, 16, hd) of 64-bit code values and scale (P, kv), in
    place, token after token."""
    x = x.double()
    P, cols = pages.shape[0], table.shape[1]
    for b in range(x.shape[0]):
        n, first = int(lengths[b]), int(positions[b])
        if not 0 <= first < cols * PAGE:
            continue
        for c in range(first // PAGE, min(cols, -(-(first + max(n, 0)) // PAGE))):
            pg = int(table[b, c])
            lo, hi = max(first - c * PAGE, 0), min(first + n - c * PAGE, PAGE)
            if not 0 <= pg < P or hi <= lo:
                continue
            t = x[b, c * PAGE + lo - first:c * PAGE + hi - first].transpose(0, 1)   # (kv, tokens, hd)
            e = exponent(torch.where(torch.isfinite(t), t, 0.0).abs().amax((1, 2)))
            if lo:
                held = torch.log2(scale[pg])
                raised = e > held
                e = torch.maximum(e, held)
                f = torch.exp2(held - e)[:, None, None]
                pages[pg, :, :lo] = torch.where(raised[:, None, None], round_e4m3(pages[pg, :, :lo] * f),
                                                pages[pg, :, :lo])
            pages[pg, :, lo:hi] = round_e4m3(t * torch.exp2(-e)[:, None, None])
            scale[pg] = torch.exp2(e)


def random_cache(pages, kv, hd, g, device="cpu", kinds=8):
    """(k, v, k_scale, v_scale) of random codes (no NaN) and scales of a few binades."""
    def codes(*shape):
        c = torch.randint(0, 127, shape, generator=g, dtype=torch.int32)
        sign = torch.randint(0, 2, shape, generator=g, dtype=torch.int32) * 128
        return (c + sign).to(torch.uint8).view(F8).to(device)

    def scale():
        return torch.exp2(torch.randint(-kinds, 1, (pages, kv), generator=g).float()).to(device)

    return codes(pages, kv, PAGE, hd), codes(pages, kv, hd, PAGE), scale(), scale()


def attention_exact(q, k, v, ks, vs, table, positions, scale):
    """q (B, n, heads, hd) over the cache in 64 bits, one (sequence, token) at a time:
    (out, sum of p |v|, largest sum of |q| |k| times scale), host tensors."""
    B, n, heads, hd = q.shape
    P, kv = ks.shape
    group = heads // kv
    out, mass = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    worst = 0.0
    for b in range(B):
        for i in range(n):
            L = min(max(int(positions[b]) + i + 1, 0), table.shape[1] * PAGE)
            at = torch.arange(L)
            pg = table[b].long()[at // PAGE] if L else at
            at, pg = at[(pg >= 0) & (pg < P)], pg[(pg >= 0) & (pg < P)]
            if not len(at):
                continue
            for j in range(kv):
                h = slice(j * group, (j + 1) * group)
                kk = k[pg, j, at % PAGE].double() * ks[pg, j, None].double()
                vv = v[pg, j, :, at % PAGE].double() * vs[pg, j, None].double()
                qq = q[b, i, h].double()
                p = torch.softmax(qq @ kk.t() * scale, 1)
                out[b, i, h] = p @ vv
                mass[b, i, h] = p @ vv.abs()
                worst = max(worst, float((qq.abs() @ kk.abs().t()).max()) * scale)
    return out, mass, worst
