"""What DecoderLayer chooses by itself, with its products and its attention replaced by ones that run on the CPU."""
import pytest
import torch as T

from project_maya_b200 import api, decoder_layer as L


class Attention:
    """Stands for api.KvAttention: keeps what it was called with."""
    def __init__(self):
        self.calls = []

    def append(self, batch, q, k, v, rope):
        self.calls.append(("append", q.dtype, k.dtype, v.dtype))
        return q

    def forward(self, batch, q, sel=None):
        self.calls.append(("forward", q.dtype))
        return q


def layer_of(cfg):
    layer = object.__new__(L.DecoderLayer)
    layer.cfg, layer.rope, layer.attn = cfg, None, Attention()
    layer.norms, layer.w_qkv, layer.w_o = {"in": T.ones(cfg.n_embd)}, None, None
    layer._product = lambda w, x, n_out: T.zeros((x.shape[0], n_out))
    return layer


@pytest.mark.parametrize("rows", [T.float32, T.bfloat16])
def test_rows_have_the_type_of_the_configuration(monkeypatch, rows):
    """Nine sequences' tokens get the bits that eight get."""
    monkeypatch.setattr(api, "_ptr", lambda t: t.data_ptr())
    cfg = L.AttentionConfig(64, 4, 2, 64, rows=rows)
    assert L.AttentionConfig(64, 4, 2, 64).rows is T.float32
    for new in ([1], [1] * 8, [1] * 9, [8], [9], [300]):
        layer = layer_of(cfg)
        out = layer.attention(T.randn((sum(new), 64)), api.AttnBatch.of(new, new, device="cpu"))
        assert layer.attn.calls == [("append", rows, rows, rows), ("forward", rows)] and out.dtype is T.float32


def test_rows_of_other_types_are_refused():
    with pytest.raises(AssertionError):
        L.AttentionConfig(64, 4, 2, 64, rows=T.float16)
