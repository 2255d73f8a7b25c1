"""What DecoderLayer does for many requests by itself - blocks reserved in front of the append, adapters beside both products - with its products and its attention
replaced by ones that run on the CPU."""
import torch as T

from project_maya_b200 import api, decoder_layer as L
from test_decoder_layer import layer_of


class Pages:
    def __init__(self, calls):
        self.calls = calls

    def reserve(self, batch):
        self.calls.append(("reserve", batch.n_tokens))


class Adapters:
    def __init__(self, name, calls):
        self.name, self.calls = name, calls

    def forward(self, x, idx, y, out=None):
        assert out is y and x.shape[0] == idx.numel() == y.shape[0]
        self.calls.append((self.name, x.shape[1], y.shape[1]))
        return y.add_(1.0)


def test_blocks_are_reserved_first_and_adapters_stand_beside_both_products(monkeypatch):
    monkeypatch.setattr(api, "_ptr", lambda t: t.data_ptr())
    cfg = L.AttentionConfig(64, 4, 2, 64)
    batch = api.AttnBatch.of([3], [3], device="cpu")
    h, idx = T.randn((3, 64)), T.tensor([0, -1, 1], dtype=T.int32)
    layer = layer_of(cfg)
    calls = layer.attn.calls
    layer.pages, layer.adapters = Pages(calls), {"qkv": Adapters("qkv", calls), "o": Adapters("o", calls)}
    out = layer.attention(h, batch, idx)
    assert [c[0] for c in calls] == ["reserve", "qkv", "append", "forward", "o"]
    assert calls[1][1:] == (64, 512) and calls[4][1:] == (256, 64) and bool((out == 1.0).all())
    layer = layer_of(cfg)
    layer.adapters = {"o": Adapters("o", layer.attn.calls)}
    layer.attention(h, batch, idx)
    assert [c[0] for c in layer.attn.calls] == ["append", "forward", "o"]
    layer = layer_of(cfg)
    layer.adapters = {"o": Adapters("o", layer.attn.calls)}
    layer.attention(h, batch)                                                      # no adapters asked for
    assert [c[0] for c in layer.attn.calls] == ["append", "forward"]
