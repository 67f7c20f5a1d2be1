"""Models whose sequences share their first KV pages: what generate and prefill refuse, before
any work on a device."""

import itertools

import pytest
import torch

from evo2_flash_amd.config import HyenaConfig
from evo2_flash_amd.model import Evo2DecodeModel

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
_number = itertools.count()  # (layer names are unique in a process)


def _model(kv_dtype, shared_prefix, B=3):
    cfg = HyenaConfig(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, intermediate_size=384, vocab_size=512,
                      hcs_layer_idxs=[0], hcm_layer_idxs=[], hcl_layer_idxs=[], attn_layer_idxs=[1])
    return Evo2DecodeModel(cfg, max_batch=B, max_ctx=64, device="cpu", kv_dtype=kv_dtype,
                           name=f"shared{next(_number)}", shared_prefix=shared_prefix)


def _prompts(B):
    return torch.zeros(B, 9, dtype=torch.int64)


@pytest.fixture
def prefilled(monkeypatch):
    """The prompts that reach the layers."""
    seen = []

    def prompts(self, tokens, chunk_seqs, layers):
        seen.append(tuple(tokens.shape))
        raise RuntimeError("reached the layers")

    monkeypatch.setattr(Evo2DecodeModel, "_prompts", prompts)
    return seen


@pytest.mark.parametrize("kv_dtype", [BF, F8])
def test_generate_refuses_prompts_that_would_share_pages(prefilled, kv_dtype):
    model = _model(kv_dtype, 32)
    for B in (2, 3):
        with pytest.raises(ValueError, match="share"):
            model.generate(_prompts(B), 3)
    assert not prefilled
    for m, B in ((model, 1), (_model(kv_dtype, 0), 3)):  # one prompt; pages of their own
        with pytest.raises(RuntimeError, match="reached"):
            m.generate(_prompts(B), 3)
    assert prefilled == [(1, 9), (3, 9)]


def test_prefill_refuses_8_bit_pages_of_several_prompts(prefilled):
    """(In bf16 pages prompts that agree on the prefix write the same values twice.)"""
    model = _model(F8, 32)
    with pytest.raises(ValueError, match="share"):
        model.prefill(_prompts(2))
    assert not prefilled
    for m, B in ((model, 1), (_model(F8, 0), 2), (_model(BF, 32), 2)):
        with pytest.raises(RuntimeError, match="reached"):
            m.prefill(_prompts(B))
    with pytest.raises(RuntimeError, match="reached"):
        model.prefill_shared(torch.zeros(32, dtype=torch.int64))
    assert prefilled == [(1, 9), (2, 9), (2, 9), (1, 32)]
