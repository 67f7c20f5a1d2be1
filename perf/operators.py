"""Cases of the training and scoring operators: attention of packed sequences with
its backward pass (`attention.packed_attention`), the gated feed-forward product with
its backward pass (`linear.gated_linear`) and the head's softmax cross entropy with
its gradient (`loss.linear_cross_entropy`).

`run` makes one call of an operator on what `prepare` gives: with `own` through the
package's entry points, else in elementary torch operations in 32 bits.  `exact`
computes the same outputs in 64 bits from the definitions.
"""

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
ACGT = (65, 67, 71, 84)
IGNORE = -100


def listed():
    return [
        # four short reads packed into one fine-tuning step, one of a single token:
        # launches and latency
        {"name": "attn_short", "op": "attn", "lens": "1,17,5,64", "heads": 32, "kv": 32,
         "hd": 128, "train": True},
        # ragged reads with shared key heads and heads of 64
        {"name": "attn_ragged", "op": "attn",
         "lens": "700,1,333,1024,65,129,511,64,800,2,255,31", "heads": 16, "kv": 4, "hd": 64,
         "train": True},
        # scoring a long prompt: no gradient
        {"name": "attn_score_8k", "op": "attn", "lens": "8192", "heads": 32, "kv": 32, "hd": 128,
         "train": False},
        # the 7B shape's attention layer in a fine-tuning step of one 8192-token sequence
        {"name": "attn_train_8k", "op": "attn", "lens": "8192", "heads": 32, "kv": 32, "hd": 128,
         "train": True},
        # a few rows through the 1B shape's MLP with GELU: the weights' bytes count
        {"name": "gated_few", "op": "gated", "rows": 5, "hidden": 1920, "inter": 5120,
         "gelu": True, "train": True},
        # the 1B shape's MLP over one 2048-token sequence
        {"name": "gated_2048", "op": "gated", "rows": 2048, "hidden": 1920, "inter": 5120,
         "gelu": True, "train": True},
        # the 7B shape's MLP over odd rows, scoring: no gradient
        {"name": "gated_score_777", "op": "gated", "rows": 777, "hidden": 4096, "inter": 11264,
         "gelu": False, "train": False},
        # the 7B shape's MLP in a fine-tuning step of 8192 tokens
        {"name": "gated_train_8k", "op": "gated", "rows": 8192, "hidden": 4096, "inter": 11264,
         "gelu": False, "train": True},
        # the likelihood of one token at the 7B shape's head
        {"name": "loss_one", "op": "loss", "rows": 1, "hidden": 4096, "vocab": 512,
         "reduction": "none", "ignored": 0.0, "train": False},
        # odd rows and an odd vocabulary, some targets ignored
        {"name": "loss_odd", "op": "loss", "rows": 777, "hidden": 1920, "vocab": 49999,
         "reduction": "none", "ignored": 0.2, "train": True},
        # the 7B shape's head in a fine-tuning step of 32768 tokens
        {"name": "loss_train_32k", "op": "loss", "rows": 32768, "hidden": 4096, "vocab": 512,
         "reduction": "mean", "ignored": 0.01, "train": True},
        # a large vocabulary, whose logits would be the step's largest tensor
        {"name": "loss_large_vocab", "op": "loss", "rows": 4096, "hidden": 4096, "vocab": 131072,
         "reduction": "mean", "ignored": 0.01, "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "gated", "loss"])
    train = rng.random() < 0.75
    if op == "attn":
        total, lens = _spread(rng, 1, 6000), []
        while total > 0:
            n = min(total, _spread(rng, 1, max(2, total)))
            lens.append(n)
            total -= n
        lens = lens[:40]
        rng.shuffle(lens)
        kv = rng.choice([1, 2, 4, 8])
        return {"op": "attn", "lens": ",".join(map(str, lens)), "heads": kv * rng.choice([1, 2, 4]),
                "kv": kv, "hd": rng.choice([64, 128]), "train": train}
    if op == "gated":
        return {"op": "gated", "rows": _spread(rng, 1, 6000), "hidden": 8 * _spread(rng, 8, 512),
                "inter": 8 * _spread(rng, 8, 1408), "gelu": rng.random() < 0.5, "train": train}
    rows = _spread(rng, 1, 8192)
    return {"op": "loss", "rows": rows, "hidden": 8 * _spread(rng, 8, 512),
            "vocab": _spread(rng, 2, min(131072, (1 << 28) // rows)),
            "reduction": rng.choice(["none", "mean", "sum"]), "ignored": rng.choice([0.0, 0.1, 0.5]),
            "train": train}


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dev=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * dev).to(BF)

    s = dict(case)
    if case["op"] == "attn":
        lens, heads, kv, hd = _lens(case), case["heads"], case["kv"], case["hd"]
        T = sum(lens)
        # queries and keys as the rotary step leaves them, values where the qkv
        # projection wrote them (a view of its rows)
        q, k = randn(T, heads, hd, dev=1.28), randn(T, kv, hd, dev=1.28)
        v = randn(T, (heads + 2 * kv) * hd, dev=1.28)[:, (heads + kv) * hd:].view(T, kv, hd)
        ends = torch.tensor([0] + lens).cumsum(0)
        s.update(q=q, k=k, v=v, cu=ends.to(torch.int32).to(DEV), scale=hd ** -0.5,
                 leaves=(q, k, v))
        if case["train"]:
            s["grad"] = randn(T, heads, hd, dev=0.01)
    elif case["op"] == "gated":
        M, H, I = case["rows"], case["hidden"], case["inter"]
        x, w1, w2 = randn(M, H), randn(I, H, dev=0.02), randn(I, H, dev=0.02)
        s.update(x=x, w1=w1, w2=w2, leaves=(x, w1, w2))
        if case["train"]:
            s["grad"] = randn(M, I, dev=0.01)
    else:
        T, H, V = case["rows"], case["hidden"], case["vocab"]
        h, w = randn(T, H), randn(V, H, dev=0.02)
        if V == 512:  # nucleotides, as bytes
            t = torch.tensor(ACGT, device=DEV)[torch.randint(4, (T,), generator=g, device=DEV)]
        else:
            t = torch.randint(V, (T,), generator=g, device=DEV)
        t = torch.where(torch.rand(T, generator=g, device=DEV) < case["ignored"], IGNORE, t)
        t[0] = min(ACGT[0], V - 1)  # the mean has a row to go by
        s.update(h=h, w=w, targets=t, leaves=(h, w))
        if case["train"]:
            # a mean or sum is the step's loss; rows of their own are weighted
            s["grad"] = (torch.rand(T, generator=g, device=DEV) if case["reduction"] == "none"
                         else torch.ones((), device=DEV))
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_()
    return s


# ------------------------------------------------------------ plain forms

def _plain_attn(s):
    q, k, v = (t.detach().float().transpose(0, 1) for t in s["leaves"])      # (heads, T, hd)
    heads, T, hd = q.shape
    kv, cu = k.shape[0], s["cu"].long()
    k, v = (t.repeat_interleave(heads // kv, 0) for t in (k, v))
    pos = torch.arange(T, device=q.device)
    seq = (pos[:, None] >= cu[None, 1:]).sum(1)
    live = (seq[:, None] == seq[None, :]) & (pos[None, :] <= pos[:, None])
    sc = torch.matmul(q, k.transpose(1, 2)) * s["scale"]
    sc = sc.masked_fill(~live, float("-inf"))
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    out = torch.matmul(p, v).transpose(0, 1).to(BF)
    if not s["train"]:
        return {"out": out}
    do = s["grad"].float().transpose(0, 1)
    dv = torch.matmul(p.transpose(1, 2), do)
    dp = torch.matmul(do, v.transpose(1, 2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(1, 2), q) * s["scale"]
    dk, dv = (t.view(kv, heads // kv, T, hd).sum(1) for t in (dk, dv))
    return {"out": out, **{n: t.transpose(0, 1).to(BF) for n, t in
                           (("dq", dq), ("dk", dk), ("dv", dv))}}


def _plain_gated(s):
    x, w1, w2 = (t.detach().float() for t in s["leaves"])
    z1, z2 = x @ w1.t(), x @ w2.t()
    if s["gelu"]:
        cdf = 0.5 * (1.0 + torch.erf(z1 * math.sqrt(0.5)))
        a = z1 * cdf
        slope = cdf + z1 * torch.exp(-0.5 * z1 * z1) / math.sqrt(2.0 * math.pi)
    else:
        a, slope = z1, torch.ones_like(z1)
    out = (a * z2).to(BF)
    if not s["train"]:
        return {"out": out}
    dh = s["grad"].float()
    d1, d2 = dh * z2 * slope, dh * a
    return {"out": out, "dx": (d1 @ w1 + d2 @ w2).to(BF), "dw1": (d1.t() @ x).to(BF),
            "dw2": (d2.t() @ x).to(BF)}


def _plain_loss(s):
    h, w = (t.detach().float() for t in s["leaves"])
    t = s["targets"]
    live = t != IGNORE
    row = torch.arange(h.shape[0], device=h.device)
    idx = torch.where(live, t, 0)
    z = h @ w.t()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    nll = torch.where(live, (top + torch.log(total)).squeeze(1) - z[row, idx], 0.0)
    count = live.sum()
    loss = {"none": nll, "sum": nll.sum(), "mean": nll.sum() / count}[s["reduction"]]
    if not s["train"]:
        return {"loss": loss}
    weight = torch.where(live, s["grad"], 0.0)
    if s["reduction"] == "mean":
        weight = weight / count
    d = e / total * weight[:, None]
    d[row, idx] -= weight
    return {"loss": loss, "dh": (d @ w).to(BF), "dw": (d.t() @ h).to(BF)}


# ------------------------------------------------------------ the package's calls

def _own_attn(s):
    from evo2_flash_amd.attention import packed_attention
    return packed_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"])


def _own_gated(s):
    from evo2_flash_amd.linear import gated_linear
    return gated_linear(s["x"], s["w1"], s["w2"], s["gelu"])


def _own_loss(s):
    from evo2_flash_amd.loss import linear_cross_entropy
    return linear_cross_entropy(s["h"], s["w"], s["targets"], ignore_index=IGNORE,
                                reduction=s["reduction"])


NAMES = {"attn": ("out", "dq", "dk", "dv"), "gated": ("out", "dx", "dw1", "dw2"),
         "loss": ("loss", "dh", "dw")}


def run(state):
    if not own:
        return {"attn": _plain_attn, "gated": _plain_gated, "loss": _plain_loss}[state["op"]](state)
    call = {"attn": _own_attn, "gated": _own_gated, "loss": _own_loss}[state["op"]]
    names = NAMES[state["op"]]
    if not state["train"]:
        with torch.no_grad():
            return {names[0]: call(state)}
    out = call(state)
    grads = torch.autograd.grad(out, state["leaves"], state["grad"])
    return {names[0]: out.detach(), **dict(zip(names[1:], grads))}


# ------------------------------------------------------------ work and 64 bits

def work(case):
    train = case["train"]
    if case["op"] == "attn":
        lens, heads, kv, hd = _lens(case), case["heads"], case["kv"], case["hd"]
        T, pairs = sum(lens), sum(n * (n + 1) // 2 for n in lens) * heads
        rows = T * hd * 2
        # scores and values; training: the products for dv, dp, dq and dk too
        return {"bytes": rows * (2 * heads + 2 * kv) + (rows * (2 * heads + 2 * kv) if train else 0),
                "flops": (12 if train else 4) * hd * pairs}
    if case["op"] == "gated":
        M, H, I = case["rows"], case["hidden"], case["inter"]
        fwd = 2 * (M * H + 2 * I * H + M * I)
        return {"bytes": fwd + (2 * (M * I + M * H + 2 * I * H) if train else 0),
                "flops": (12 if train else 4) * M * H * I}
    T, H, V = case["rows"], case["hidden"], case["vocab"]
    fwd = 2 * (T * H + V * H) + 8 * T + (4 * T if case["reduction"] == "none" else 4)
    back = 2 * (T * H + V * H) + (4 * T if case["reduction"] == "none" else 4)
    return {"bytes": fwd + (back if train else 0), "flops": (6 if train else 2) * T * H * V}


def _exact_attn(case, s):
    q, k, v = (t.detach().double() for t in s["leaves"])
    do = s["grad"].double() if case["train"] else None
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    group, at = case["heads"] // case["kv"], 0
    for n in _lens(case):
        r = slice(at, at + n)
        at += n
        tri = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(case["heads"]):
            j = h // group
            p = torch.softmax(((q[r, h] * s["scale"]) @ k[r, j].t()).masked_fill(tri, -math.inf), 1)
            out[r, h] = p @ v[r, j]
            if do is not None:
                dv[r, j] += p.t() @ do[r, h]
                # the softmax's own gradient, p (dp - p . dp)
                dp = do[r, h] @ v[r, j].t()
                ds = p * dp
                ds = (ds - p * ds.sum(1, keepdim=True)) * s["scale"]
                if n == 1:  # one key: its probability is 1 whatever the score
                    ds.zero_()
                dq[r, h] = ds @ k[r, j]
                dk[r, j] += ds.t() @ q[r, h]
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"out": out}


def _exact_gated(case, s):
    x, w1, w2 = (t.detach().double().requires_grad_() for t in s["leaves"])
    z1 = torch.nn.functional.linear(x, w1)
    if case["gelu"]:
        z1 = torch.nn.functional.gelu(z1)
    out = z1 * torch.nn.functional.linear(x, w2)
    if not case["train"]:
        return {"out": out.detach()}
    grads = torch.autograd.grad(out, (x, w1, w2), s["grad"].double())
    return {"out": out.detach(), **dict(zip(NAMES["gated"][1:], grads))}


def _exact_loss(case, s):
    h, w = (t.detach().double().requires_grad_() for t in s["leaves"])
    loss = torch.nn.functional.cross_entropy(torch.nn.functional.linear(h, w), s["targets"],
                                             ignore_index=IGNORE, reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss.detach()}
    grads = torch.autograd.grad(loss, (h, w), s["grad"].double())
    return {"loss": loss.detach(), **dict(zip(NAMES["loss"][1:], grads))}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "gated": _exact_gated, "loss": _exact_loss}[case["op"]](case, s)
