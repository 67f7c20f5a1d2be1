"""The decoder with its KV pages in 8 bits, and generation: the operators together, as a user
runs them.

* prefill leaves the pages that quantising a bf16 model's pages gives, bit for bit (the layers
  below an attention layer are the same ones), and the same logits;
* each decode step's attention layer against fp32 attention over the values of a cache written
  from the layer's own keys and values: within the bf16 composition's 2e-2;
* generate draws what sample_tokens draws from the steps' logits, with either type of pages;
* the whole step with the draw, captured once, replays like eager steps."""

import itertools

import pytest
import torch

from evo2_flash_amd.attention import PAGE, PagedKVCache, rotary_decode
from evo2_flash_amd.config import HyenaConfig
from evo2_flash_amd.kv_fp8 import Fp8KVCache
from evo2_flash_amd.model import Evo2DecodeModel
from evo2_flash_amd.sampling import sample_tokens

from _cases import max_rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
SHAPES = [(256, 4), (512, 4)]  # heads of 64 and 128
_number = itertools.count()    # (layer names are unique in a process)


def _model(H, heads, kv_dtype, B=3, ctx=96, **kw):
    cfg = HyenaConfig(hidden_size=H, num_hidden_layers=5, num_attention_heads=heads,
                      intermediate_size=384, vocab_size=512, hcs_layer_idxs=[0, 4],
                      hcm_layer_idxs=[1], hcl_layer_idxs=[2], attn_layer_idxs=[3],
                      use_fp8_input_projections=True)
    m = Evo2DecodeModel(cfg, max_batch=B, max_ctx=ctx, device=DEV, rope_factor=4.0,
                        name=f"generate{next(_number)}", kv_dtype=kv_dtype, **kw)
    return m.init_random(seed=21, state_scale=0.0, kv_scale=0.0)


def _bytes(cache):
    return [t.view(torch.uint8) for t in cache.tensors]


@pytest.mark.parametrize("H,heads", SHAPES)
@pytest.mark.parametrize("L", [1, 16, 37])
def test_prefill_writes_the_quantised_pages(H, heads, L):
    a, b = _model(H, heads, F8), _model(H, heads, torch.bfloat16)
    g = torch.Generator().manual_seed(L)
    tokens = torch.randint(512, (3, L), generator=g).to(DEV)
    assert torch.equal(a.prefill(tokens), b.prefill(tokens))
    got, plain = a.layers[3].mixer.cache, b.layers[3].mixer.cache
    want = Fp8KVCache(plain.k.shape[0], heads, H // heads, DEV)
    k, v = plain.dense(b.block_table, 3, L)
    want.write_prompt(k.transpose(2, 3), v, b.block_table)
    for x, y in zip(_bytes(got), _bytes(want)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("H,heads", SHAPES)
def test_decode_attention_layer(H, heads):
    model, hd = _model(H, heads, F8), H // heads
    a = model.layers[3].mixer
    shadow = Fp8KVCache(a.cache.k.shape[0], heads, hd, DEV)
    scratch = PagedKVCache(a.cache.k.shape[0], heads, hd, DEV)
    g = torch.Generator().manual_seed(1)
    table, b = model.block_table, torch.arange(3, device=DEV)
    for step in range(40):
        x = torch.randn(3, H, generator=g).to(torch.bfloat16).to(DEV)
        pos = torch.tensor([step, step + 20, step], device=DEV)
        got = a.forward_decode(x, pos, table)
        qkv, _ = a.qkv_proj(x)
        q = rotary_decode(qkv, scratch, table, pos, a.inv_freq, a.rope_factor)
        page = table[b, pos // PAGE].long()
        shadow.append(scratch.k[page, :, :, pos % PAGE], scratch.v[page, :, pos % PAGE], table, pos)
        for x1, y1 in zip(_bytes(a.cache), _bytes(shadow)):
            assert torch.equal(x1, y1), step
        k, v = shadow.dense(table, 3, 96)
        s = (q.float()[:, :, None] @ k.float())[:, :, 0] * hd ** -0.5
        s = s.masked_fill(torch.arange(96, device=DEV) > pos[:, None, None], float("-inf"))
        out = (torch.softmax(s, 2)[:, :, None] @ v.float())[:, :, 0].to(torch.bfloat16)
        want, _ = a.o_proj(out.reshape(3, H))
        assert max_rel_err(got.cpu(), want.cpu()) <= 2e-2, step


@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, F8])
@pytest.mark.parametrize("H,heads", SHAPES)
def test_generate_draws_from_the_steps_logits(H, heads, kv_dtype):
    model = _model(H, heads, kv_dtype)
    g = torch.Generator().manual_seed(2)
    prompts = torch.randint(512, (3, 29), generator=g).to(DEV)
    u = torch.rand(24, 3, generator=g).to(DEV)
    settings = dict(temperature=torch.tensor([1.0, 0.7, 0.0], device=DEV), top_k=50, top_p=0.9,
                    min_p=0.01)
    got = model.generate(prompts, 24, uniforms=u, **settings)
    assert got.shape == (3, 24) and int(got.min()) >= 0 and int(got.max()) < 512
    logits = model.prefill(prompts)
    for i in range(24):
        tok = sample_tokens(logits, u[i], **settings)
        assert torch.equal(got[:, i], tok), i
        logits = model.decode_step(tok, torch.full((3,), 29 + i, device=DEV))
    assert torch.equal(model.generate(prompts, 24, uniforms=u, **settings), got)
    a = model.generate(prompts[:2], 5, generator=torch.Generator(device=DEV).manual_seed(3))
    b = model.generate(prompts[:2], 5, generator=torch.Generator(device=DEV).manual_seed(3))
    assert torch.equal(a, b) and a.shape == (2, 5)
    assert model.generate(prompts, 0).shape == (3, 0)
    with pytest.raises(ValueError, match="exceed"):
        model.generate(prompts, 96 - 29 + 2)
    with pytest.raises(ValueError, match="uniforms"):
        model.generate(prompts, 3, uniforms=u)
    with pytest.raises(ValueError, match="at least one"):
        model.generate(prompts[:, :0], 3)


def test_rows_of_nan_logits_draw_no_token():
    model = _model(256, 4, F8)
    model.norm.weight.data.fill_(float("nan"))
    got = model.generate(torch.ones(2, 9, dtype=torch.int64, device=DEV), 3)
    assert got.tolist() == [[-1] * 3] * 2


@pytest.mark.parametrize("H,heads", SHAPES)
def test_step_with_the_draw_in_a_graph(H, heads):
    a, b = _model(H, heads, F8), _model(H, heads, F8)
    g = torch.Generator().manual_seed(4)
    prompts = torch.randint(512, (3, 20), generator=g).to(DEV)
    tok, pos = torch.zeros(3, dtype=torch.int64, device=DEV), torch.full((3,), 20, device=DEV)
    u = torch.zeros(3, device=DEV)

    def step(model):
        return sample_tokens(model.decode_step(tok, pos), u, 0.9, 40, 0.95)

    a.prefill(prompts)
    step(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    a.prefill(prompts)
    b.prefill(prompts)
    for x, y in zip(_bytes(a.layers[3].mixer.cache), _bytes(b.layers[3].mixer.cache)):
        x.copy_(y)  # (pages past the prompt: the warm-up's token)
    for i in range(30):
        u.copy_(torch.rand(3, generator=g))
        pos.fill_(20 + i)
        want = step(b)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(out, want), i
        tok.copy_(want)


def test_shared_prefix_and_a_long_context():
    """Sequences behind a shared prompt, their own pages behind it: the declared pages give
    what undeclared ones do, within a rounding step of the logits' arithmetic."""
    model = _model(512, 4, F8, B=5, ctx=160, shared_prefix=96)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(512, (96,), generator=g).to(DEV)
    model.prefill_shared(prompt)
    a = model.layers[3].mixer
    assert a.shared_pages == 6
    x = torch.randn(5, 512, generator=g).to(torch.bfloat16).to(DEV)
    pos = torch.full((5,), 96, device=DEV)
    one = a.forward_decode(x, pos, model.block_table)
    a.shared_pages = 0
    two = a.forward_decode(x, pos, model.block_table)
    assert max_rel_err(one.cpu(), two.cpu()) <= 2e-2
    assert model.decode_step(torch.randint(512, (5,), generator=g).to(DEV), pos + 1).shape == (5, 512)


def test_random_pages():
    model = _model(256, 4, F8)
    model.init_random(seed=3, kv_scale=0.5)
    k, v = model.layers[3].mixer.cache.dense(model.block_table, 3, 96)
    for t in (k, v):
        assert 0.45 < float(t.float().std()) < 0.55 and torch.isfinite(t).all()
    model.init_random(seed=3, kv_scale=0.0)
    assert not model.layers[3].mixer.cache.k.view(torch.uint8).any()
