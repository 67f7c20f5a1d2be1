"""The training operators' refusals, without a GPU: the wrappers' checks on CPU tensors
(the device check apart) and the C entries' argument checks, which come before any
launch; the plan of work queries."""

import pytest
import torch

from evo2_flash_amd import _lib
from evo2_flash_amd.attention import packed_attention
from evo2_flash_amd.linear import gated_linear
from evo2_flash_amd.loss import linear_cross_entropy

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        packed_attention(_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), torch.tensor([0, 4]), 0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_linear(_z(4, 8), _z(8, 8), _z(8, 8), False)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_cross_entropy(_z(4, 8), _z(8, 8), torch.zeros(4, dtype=torch.int64))


@pytest.fixture
def native(monkeypatch):
    """CPU tensors pass the device check; a call is an error."""
    def call(name, *args):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(_lib, "call", call)


CU = torch.tensor([0, 4])


@pytest.mark.parametrize("q,k,v,cu,scale,match", [
    (_z(4, 128), _z(4, 2, 64), _z(4, 2, 64), CU, 0.1, "takes bf16 q"),
    (_z(4, 2, 64, dtype=torch.float16), _z(4, 2, 64), _z(4, 2, 64), CU, 0.1, "takes bf16 q"),
    (_z(4, 2, 64), _z(5, 2, 64), _z(5, 2, 64), CU, 0.1, "do not match"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 1, 64), CU, 0.1, "do not match"),
    (_z(4, 3, 64), _z(4, 2, 64), _z(4, 2, 64), CU, 0.1, "do not match"),
    (_z(4, 2, 64), _z(4, 0, 64), _z(4, 0, 64), CU, 0.1, "do not match"),
    (_z(4, 2, 80), _z(4, 2, 80), _z(4, 2, 80), CU, 0.1, "head_dim 64 or 128"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), CU[:0], 0.1, "cu_seqlens must be"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), CU.float(), 0.1, "cu_seqlens must be"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), CU[None], 0.1, "cu_seqlens must be"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), CU, 0.0, "positive scale"),
    (_z(4, 2, 64), _z(4, 2, 64), _z(4, 2, 64), CU, float("inf"), "positive scale"),
])
def test_packed_attention_refuses(native, q, k, v, cu, scale, match):
    with pytest.raises(ValueError, match=match):
        packed_attention(q, k, v, cu, scale)


@pytest.mark.parametrize("x,w1,w2,match", [
    (_z(4, 8, dtype=torch.float32), _z(8, 8), _z(8, 8), "takes bf16"),
    (_z(4, 8), _z(8, 8), _z(16, 8), "do not match"),
    (_z(4, 16), _z(8, 8), _z(8, 8), "do not match"),
    (_z(4, 8), _z(2, 8, 8), _z(2, 8, 8), "do not match"),
    (_z(4, 8), _z(12, 8), _z(12, 8), "multiples of 8"),
    (_z(4, 12), _z(8, 12), _z(8, 12), "multiples of 8"),
    (_z(4, 8), _z(0, 8), _z(0, 8), "multiples of 8"),
])
def test_gated_linear_refuses(native, x, w1, w2, match):
    with pytest.raises(ValueError, match=match):
        gated_linear(x, w1, w2, False)


T4 = torch.zeros(4, dtype=torch.int64)


@pytest.mark.parametrize("h,w,t,red,match", [
    (_z(4, 8), _z(9, 8), T4, "average", "reduction must be"),
    (_z(4, 8, dtype=torch.float32), _z(9, 8), T4, "mean", "takes bf16"),
    (_z(4, 16), _z(9, 8), T4, "mean", "do not match"),
    (_z(4, 8), _z(9, 8), T4[:3], "mean", "do not match"),
    (_z(4, 8), _z(9, 8), T4.view(2, 2), "mean", "do not match"),
    (_z(4, 12), _z(9, 12), T4, "mean", "multiple of 8"),
    (_z(4, 8), _z(0, 8), T4, "mean", "at least one row"),
    (_z(4, 8), _z(9, 8), T4.float(), "mean", "integers"),
])
def test_linear_cross_entropy_refuses(native, h, w, t, red, match):
    with pytest.raises(ValueError, match=match):
        linear_cross_entropy(h, w, t, reduction=red)


INVALID, UNSUPPORTED = 1, 2


def test_c_entries_check_before_a_launch():
    lib, n, at = _lib.lib(), None, 4096  # (an aligned address that is never read)

    def attention(T=8, nseq=1, heads=4, kv=2, hd=64, scale=0.1, q=at, sq=256, lo=n, lse=n):
        return lib.evo2_packed_attention(q, sq, 64, at, 128, 64, at, 128, 64, at, nseq, at, lo, lse,
                                         T, heads, kv, hd, scale, n)

    assert attention(T=0) == 0
    assert attention(kv=3) == INVALID and attention(T=-1) == INVALID
    assert attention(scale=-1.0) == INVALID and attention(scale=float("nan")) == INVALID
    assert attention(hd=96) == UNSUPPORTED
    assert attention(q=n) == INVALID and attention(lo=at) == INVALID
    assert attention(q=at + 2) == UNSUPPORTED and attention(sq=252) == UNSUPPORTED
    assert attention(sq=56) == UNSUPPORTED  # overlapping rows
    assert attention(sq=1 << 23) == UNSUPPORTED
    need = lib.evo2_packed_attention_workspace_bytes(8, 1, 4, 2, 64)
    assert need == 256 + 4 * 8 * 2 * 64 * 4
    assert lib.evo2_packed_attention_workspace_bytes(8, 1, 4, 4, 64) == 256
    rc = lib.evo2_packed_attention_backward(at, 256, 64, at, 256, 64, at, 128, 64, at, 128, 64, at, 1,
                                            at, at, at, at, need - 1, at, at, at, 8, 4, 2, 64, 0.1, n)
    assert rc == INVALID and b"workspace" in lib.evo2_last_error()

    def gated(M=4, I=16, H=8, sx=8, x=at):
        return lib.evo2_gated_linear(x, sx, at, at, 8, 0, at, 16, n, M, I, H, n)

    assert gated(M=0) == 0
    assert gated(M=-1) == INVALID and gated(I=0) == INVALID and gated(x=n) == INVALID
    assert gated(I=12) == UNSUPPORTED and gated(H=4) == UNSUPPORTED
    assert gated(sx=4) == UNSUPPORTED and gated(x=at + 8) == UNSUPPORTED
    assert gated(I=1 << 31) == UNSUPPORTED
    need = lib.evo2_gated_linear_workspace_bytes(4, 16, 8)

    def gated_back(M=4, dw2=at, bytes=need):
        return lib.evo2_gated_linear_backward(at, 16, at, 8, at, at, 8, at, at, at, dw2, at, bytes, M,
                                              16, 8, n)

    assert gated_back(M=0) == INVALID and gated_back(dw2=n) == INVALID
    assert gated_back(bytes=need - 1) == INVALID and b"workspace" in lib.evo2_last_error()

    def loss(T=4, V=9, H=8, red=2, out=at, sh=8, bytes=1 << 20):
        return lib.evo2_linear_loss(at, sh, at, 8, at, -100, red, at, at, out, out, at, bytes, T, V, H, n)

    assert loss(T=0) == INVALID and loss(V=0) == INVALID and loss(red=3) == INVALID
    assert loss(out=n) == INVALID and loss(H=12) == UNSUPPORTED and loss(sh=4) == UNSUPPORTED
    assert loss(bytes=16) == INVALID and b"workspace" in lib.evo2_last_error()
    rc = lib.evo2_linear_loss_backward(at, 8, at, 8, at, -100, at, at, 1, at, at, at, at, 1 << 20, 4, 9,
                                       8, n)
    assert rc == INVALID  # a mean's upstream gradient is one value


@pytest.mark.parametrize("T,V,H", [(1, 512, 4096), (777, 49999, 1920), (32768, 512, 4096),
                                   (4096, 131072, 4096), (17000, 9000, 16), (5, 3, 8)])
def test_loss_workspaces_keep_no_logits(T, V, H):
    """Forward: partial logits of at most a card of tiles, or 16 bytes a row for every 256
    columns; backward: d in pieces of 256 MB (or 8192 columns) and fp32 sums."""
    lib = _lib.lib()
    forward, back = (lib.evo2_linear_loss_workspace_bytes(T, V, H, b) for b in (0, 1))
    assert 0 < forward <= max(256 * 256 * 256 * 4, T * -(-V // 256) * 16 + 4 * T) + 64 * T + 4096
    d = T * min(V + 8, max(8192, (1 << 27) // T)) * 2
    assert 0 < back <= d + T * H * 4 + 8 * 256 * 256 * 256 + 4096


def test_score_and_training_are_the_models():
    from evo2_flash_amd.model import Evo2DecodeModel, Evo2DecoderLayer

    assert callable(Evo2DecodeModel.score) and callable(Evo2DecodeModel.training_loss)
    layer = Evo2DecoderLayer.__new__(Evo2DecoderLayer)
    torch.nn.Module.__init__(layer)
    layer.kind = "hcl"
    with pytest.raises(NotImplementedError, match="Hyena"):
        layer.forward_train(torch.zeros(1, 8), None, None)
