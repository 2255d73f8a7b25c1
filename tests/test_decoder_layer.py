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


def test_each_sequence_reads_selected_blocks_by_its_own_length(monkeypatch):
    """What a short context's token reads must not depend on a long one beside it."""
    monkeypatch.setattr(api, "_ptr", lambda t: t.data_ptr())

    class Counting(Attention):
        def forward(self, batch, q, sel=None):
            if sel is None:
                assert int(batch.kv_len.max()) <= batch.desc.max_len          # (lengths beyond the bound would be cut)
            seen = batch.kv_len.view(-1, 1, 1) * (1 if sel is None else 1000)
            return seen.expand(-1, *q.shape[1:]).to(q.dtype)

        def select(self, batch, q):
            return "list"

    cfg = L.AttentionConfig(64, 4, 2, 64, n_sel=4, sparse_from=100)
    for lens in ([700], [99], [99, 100], [5000, 7, 99, 101], [100, 2000]):
        for batch in (api.AttnBatch.of([1] * len(lens), lens, device="cpu"),
                      api.AttnBatch(T.arange(len(lens) + 1, dtype=T.int32), T.tensor(lens, dtype=T.int32), len(lens), 1, 9999)):
            layer = layer_of(cfg)
            layer.attn = Counting()
            out = layer._attend(batch, T.zeros((len(lens), 4, 64)))
            assert out[:, 0, 0].tolist() == [n if n < 100 else 1000 * n for n in lens]
    window = api.AttnBatch.of([2], [700], device="cpu")                        # more than a token: every block
    assert layer._attend(window, T.zeros((1, 4, 64)))[0, 0, 0] == 700
