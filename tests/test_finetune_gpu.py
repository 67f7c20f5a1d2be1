"""The decoder harness's scoring and training paths (model.score,
model.training_loss) against the same weights in plain torch: log-likelihoods from
the logits of a prefill, and loss and gradients of the layers above the last Hyena
mixer from autograd in 64 bits on the same features.

The training path rounds activations to bf16 at every operator: some twenty roundings
of u = 2^-8 each lie between a parameter and the loss.  Independent, they add up to
about sqrt(20) u / sqrt(3) of a gradient's norm, 1%; the checks allow 3%."""

import pytest
import torch

from evo2_flash_amd.config import HyenaConfig
from evo2_flash_amd.model import Evo2DecodeModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACGT = [65, 67, 71, 84]


def _model(H, heads, name, max_batch=3, max_ctx=160, attn=(1, 3, 4)):
    kinds = {"hcs_layer_idxs": [0], "hcl_layer_idxs": [2], "attn_layer_idxs": list(attn)}
    cfg = HyenaConfig(hidden_size=H, num_hidden_layers=5, num_attention_heads=heads,
                      intermediate_size=384, vocab_size=512, use_fp8_input_projections=True, **kinds)
    m = Evo2DecodeModel(cfg, max_batch=max_batch, max_ctx=max_ctx, device=DEV, rope_theta=10000.0,
                        rope_factor=2.0, name=name, page_seed=1)
    return m.init_random(seed=3, state_scale=0.0, kv_scale=0.0, embed_scale=0.5)


def _tokens(B, L, seed=4):
    g = torch.Generator().manual_seed(seed)
    return torch.tensor(ACGT)[torch.randint(0, 4, (B, L), generator=g)].to(DEV)


@pytest.mark.parametrize("L", [1, 2, 37, 130])
def test_score_is_the_logits_log_likelihood(L):
    model, tok = _model(256, 4, f"score{L}"), _tokens(3, L)
    print(f"score 3 x {L}", flush=True)
    got = model.score(tok, chunk_seqs=2)
    assert got.shape == (3, L - 1) and got.dtype == torch.float32
    for n in sorted({1, L // 2, L - 1} & set(range(1, L))):
        logits = model.prefill(tok[:, :n]).double()  # bf16: u of logits up to ~40
        want = torch.log_softmax(logits, 1).gather(1, tok[:, n:n + 1])[:, 0]
        # two prompts of different lengths: their features differ by bf16 roundings
        assert (got[:, n - 1].double() - want).abs().max() <= 2e-2 * logits.abs().max(), (L, n)


def _reference(model, x, targets, B, L):
    """(loss, {name: gradient}) of the layers above the features x in 64 bits."""
    ps = {n: p.detach().double().cpu().requires_grad_() for n, p in model.named_parameters()
          if p.requires_grad}

    def get(mod, attr, prefix):
        p = getattr(mod, attr)
        return None if p is None else ps.get(prefix + attr, p.detach().double().cpu())

    def norm(mod, v, prefix):
        w = get(mod, "weight", prefix)
        return w * v / (v.norm(dim=-1, keepdim=True) * v.shape[-1] ** -0.5 + mod.eps)

    x = x.detach().double().cpu()
    F = torch.nn.functional
    first = len(model.layers) - len(model.trained_layers())
    for i, layer in enumerate(model.trained_layers(), first):
        p, a = f"layers.{i}.", layer.mixer
        h = norm(layer.pre_norm, x, p + "pre_norm.")
        q, k, v = F.linear(h, get(a.qkv_proj, "weight", p + "mixer.qkv_proj.")).view(
            B, L, 3, a.heads, a.hd).permute(2, 0, 3, 1, 4)
        ang = (torch.arange(L).double() / a.rope_factor)[:, None] * a.inv_freq.double().cpu()

        def rot(t):
            t1, t2 = t.chunk(2, -1)
            return torch.cat([t1 * ang.cos() - t2 * ang.sin(), t2 * ang.cos() + t1 * ang.sin()], -1)

        s = rot(q) @ rot(k).transpose(-1, -2) * a.hd ** -0.5
        s = s.masked_fill(torch.ones(L, L, dtype=torch.bool).triu(1), float("-inf"))
        o = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * L, -1)
        x = x + F.linear(o, get(a.o_proj, "weight", p + "mixer.o_proj."),
                         get(a.o_proj, "bias", p + "mixer.o_proj."))
        h, m = norm(layer.post_norm, x, p + "post_norm."), layer.mlp
        z = F.linear(h, get(m.l1, "weight", p + "mlp.l1."))
        z = (F.gelu(z) if m.use_act else z) * F.linear(h, get(m.l2, "weight", p + "mlp.l2."))
        x = x + F.linear(z, get(m.l3, "weight", p + "mlp.l3."))
    h = norm(model.norm, x, "norm.")
    loss = F.cross_entropy(F.linear(h, get(model, "embed", "")), targets.reshape(-1).cpu())
    return loss.detach(), dict(zip(ps, torch.autograd.grad(loss, list(ps.values()),
                                                           allow_unused=True)))


@pytest.mark.parametrize("heads,L", [(4, 61), (2, 129)])
def test_training_loss_and_gradients(heads, L):
    """Two attention layers above the last Hyena mixer, heads of 64 and 128; padded
    targets; parameters below get no gradient."""
    model, tok = _model(256, heads, f"train{L}"), _tokens(3, L)
    top = model.trained_layers()
    assert [layer.kind for layer in top] == ["attn", "attn"]
    for layer in top:
        layer.requires_grad_()
    model.embed.requires_grad_()
    targets = torch.full_like(tok, -100)
    targets[:, :-1] = tok[:, 1:]
    targets[1, L // 2:] = -100
    print(f"training_loss 3 x {L}, {heads} heads", flush=True)
    loss = model.training_loss(tok, targets, chunk_seqs=2)
    loss.backward()
    with torch.no_grad():
        x = torch.cat([r for _, _, r in model._prompts(tok, 2, model.layers[:3])])
    want, grads = _reference(model, x, targets, 3, L)
    assert abs(loss.item() - want.item()) <= 3e-2 * abs(want.item())
    for n, p in model.named_parameters():
        if n.startswith(("layers.0.", "layers.1.", "layers.2.")):
            assert p.grad is None, n
        elif p.requires_grad:
            off = (p.grad.double().cpu() - grads[n]).norm() / grads[n].norm()
            assert off <= 3e-2, (n, off.item())
    assert model.training_loss(tok, chunk_seqs=3).item() != loss.item()  # unpadded targets


def test_layers_with_hooks_and_hyena_layers():
    model, tok = _model(256, 4, "train_hooks"), _tokens(2, 20)
    mlp = model.trained_layers()[0].mlp
    mlp.l1.weight.requires_grad_()
    seen = []
    plain = model.training_loss(tok)
    handle = mlp.l1.register_forward_hook(lambda m, a, out: seen.append(out[0].shape))
    hooked = model.training_loss(tok)
    handle.remove()
    assert seen == [torch.Size([40, 384])]
    assert abs(plain.item() - hooked.item()) <= 1e-2 * abs(plain.item())
    with pytest.raises(NotImplementedError, match="Hyena"):
        model.layers[0].forward_train(torch.zeros(4, 256, device=DEV), None, None)


def test_training_under_compile_and_checkpoints():
    """The operators inside a compiled function, a checkpointed one and autocast give the
    eager bits; forward-mode tangents, which they have not, are refused."""
    from torch.utils.checkpoint import checkpoint

    from evo2_flash_amd.attention import packed_attention
    from evo2_flash_amd.linear import gated_linear
    from evo2_flash_amd.loss import linear_cross_entropy

    g = torch.Generator().manual_seed(6)

    def leaf(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16).to(DEV).requires_grad_()

    q, k, v = (leaf(40, 2, 64) for _ in range(3))
    w1, w2 = leaf(72, 128), leaf(72, 128)
    cu = torch.tensor([0, 15, 40], dtype=torch.int32, device=DEV)
    t = torch.randint(72, (40,), generator=g).to(DEV)
    leaves = (q, k, v, w1, w2)

    def f(q, k, v, w1, w2):
        x = packed_attention(q, k, v, cu, 0.1).view(40, 128)
        return linear_cross_entropy(x, w1, t) + gated_linear(x, w1, w2, True).float().mean()

    want = f(*leaves)
    grads = torch.autograd.grad(want, leaves)

    def same(loss):
        got = torch.autograd.grad(loss, leaves)
        return torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(got, grads))

    assert same(torch.compile(f)(*leaves))
    assert same(checkpoint(f, *leaves, use_reentrant=False))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = f(*leaves)
    assert same(loss)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.detach(), torch.ones_like(q))
        with pytest.raises(Exception, match="jvp"):
            packed_attention(dual, k.detach(), v.detach(), cu, 0.1)


def test_other_sizes_take_the_modules():
    """An MLP off the operator's sizes trains through its modules."""
    from evo2_flash_amd.model import Evo2MLP

    mlp = Evo2MLP(64, 36, True, device=DEV).requires_grad_()
    for m in (mlp.l1, mlp.l2, mlp.l3):
        torch.nn.init.normal_(m.weight, std=0.1)
    x = torch.randn(5, 64, device=DEV).to(torch.bfloat16)
    out = mlp.forward_train(x)
    assert torch.equal(out, mlp(x))
    out.sum().backward()
    assert all(m.weight.grad.isfinite().all() for m in (mlp.l1, mlp.l2, mlp.l3))
