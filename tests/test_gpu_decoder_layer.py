"""A whole decoder layer: the attention half (GGUF products, norms, rotation, 8-bit cache, attention) in front of the experts, over a prompt, a window and
single tokens, against the same attention written out over dequantized weights."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def layer_of(n_sel=0, sparse_from=8192, tokens=400):
    from project_maya_b200 import api, decoder_layer as L
    cfg = L.AttentionConfig(512, 8, 2, 64, n_sel=n_sel, sparse_from=sparse_from)
    return L.synthetic_layer(cfg, api.MoeLayerConfig(512, 256, 8, 2, api.Q8_0, api.Q8_0), tokens, 512)


def dequantize_q8_0(raw, rows, cols):
    b = raw.cpu().numpy().reshape(rows, cols // 32, 34)
    d = b[:, :, :2].copy().view(np.float16).astype(np.float64)
    return (b[:, :, 2:].view(np.int8) * d).reshape(rows, cols)


def plain_attention(layer, h):
    """The attention half over all tokens of one sequence in 64 bits, nothing rounded."""
    c, n = layer.cfg, {k: v.double().cpu().numpy() for k, v in layer.norms.items()}
    rms = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + c.eps) * w   # noqa: E731
    rows = rms(h, n["in"]) @ dequantize_q8_0(layer.w_qkv, c.qkv_rows, c.n_embd).T
    q, k, v = np.split(rows.reshape(len(h), -1, c.head_dim), (c.n_q, c.n_q + c.n_kv), 1)
    half = c.head_dim // 2
    angle = np.arange(len(h))[:, None, None] * c.theta ** (-np.arange(half) / half)

    def turn(x):
        a, b = x[..., :half], x[..., half:]
        return np.concatenate((a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)), -1)

    q, k = turn(rms(q, n["q"])), turn(rms(k, n["k"]))
    g = c.n_q // c.n_kv
    s = np.einsum("ihd,jhd->hij", q, np.repeat(k, g, 1)) / np.sqrt(c.head_dim)
    s[:, ~np.tri(len(h), dtype=bool)] = -np.inf
    p = np.exp(s - s.max(-1, keepdims=True))
    o = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), np.repeat(v, g, 1))
    return o.reshape(len(h), -1) @ dequantize_q8_0(layer.w_o, c.n_embd, c.n_q * c.head_dim).T


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def test_attention_half_over_prompt_window_and_tokens(cuda):
    """8-bit activations of both products, 8-bit keys and values: each rounds by amax / 254 a value, of values of some 1/3 to 1/4 of amax rms - 1 % apart, so
    within 4 % all together."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(5)
    layer, n = layer_of(), 300
    h = T.randn((n, 512), device="cuda")
    want = plain_attention(layer, h.double().cpu().numpy())
    got, at = [], 0
    for new in (130, 64, 20, 9, 7, 1, 1, 3, *[1] * 5, 60):                     # chunks by the GEMM, windows and tokens by the GEMV
        got.append(layer.attention(h[at:at + new], api.AttnBatch.of([new], [at + new])))
        at += new
    assert at == n
    got = T.cat(got).double().cpu().numpy()
    assert rel(got, want) < 0.04
    assert max(rel(got[i], want[i]) for i in range(n)) < 0.15                  # no row is wrong (few tokens' rows round more)
    assert layer.attn.error() == 0


def test_layer_prompt_equals_tokens(cuda):
    """The whole layer: a prompt at once and token by token end in like outputs (routing may differ where two experts' scores are near)."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(6)
    h = T.randn((70, 512), device="cuda")
    a, b = layer_of(), layer_of()
    whole = a.forward(h, api.AttnBatch.of([70], [70]))
    single = T.cat([b.forward(h[i:i + 1], api.AttnBatch.of([1], [i + 1])) for i in range(70)])
    err = ((whole - single).norm(dim=1) / single.norm(dim=1)).cpu().numpy()
    assert np.median(err) < 0.02 and np.isfinite(err).all()


def test_layer_with_selected_blocks(cuda):
    """A long context through select(): with as many entries as blocks the same as without; with fewer, the lists' blocks alone."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(7)
    h = T.randn((400, 512), device="cuda")
    outs = []
    for n_sel in (0, 7, 4):
        layer = layer_of(n_sel=n_sel, sparse_from=1)
        layer.attention(h[:399], api.AttnBatch.of([399], [399]))
        outs.append(layer.attention(h[399:], api.AttnBatch.of([1], [400])).double().cpu().numpy())
    assert rel(outs[1], outs[0]) < 1e-3                                        # (sums in another order, rounded to 8 bits once more)
    assert 1e-3 < rel(outs[2], outs[0]) < 1.0


def test_short_contexts_beside_long_ones_read_every_block(cuda):
    """A batch of a context beyond `sparse_from` and one below it: the short one's token is what it is without selection, the long one's what it is alone."""
    import torch as T
    from project_maya_b200 import api, decoder_layer as L
    T.manual_seed(8)
    lens = (400, 330)
    h = [T.randn((n, 512), device="cuda") for n in lens]

    def run(n_sel, which, batch_of=api.AttnBatch.of):
        cfg = L.AttentionConfig(512, 8, 2, 64, n_sel=n_sel, sparse_from=350)
        layer = L.synthetic_layer(cfg, api.MoeLayerConfig(512, 256, 8, 2, api.Q8_0, api.Q8_0), 400, 512, n_seq=2)
        layer.attention(T.cat([x[:-1] for x in h]), api.AttnBatch.of([n - 1 for n in lens], [n - 1 for n in lens]))
        out = layer.attention(T.cat([h[i][-1:] for i in which]), batch_of([int(i in which) for i in (0, 1)], lens))
        assert layer.attn.error() == 0
        return out.double().cpu().numpy()

    def bounds_alone(new, kv_len):                                             # as a graph's batch: lengths on the device, a bound on the host
        b = api.AttnBatch.of(new, kv_len)
        return api.AttnBatch(b.start, b.kv_len, b.n_tokens, 1, 400)

    both, dense, alone = run(4, (0, 1)), run(0, (0, 1)), run(4, (0,))
    assert rel(both[1], dense[1]) < 1e-3 and rel(both[0], alone[0]) < 1e-3     # (sums in another order, rounded to 8 bits once more)
    assert rel(both[0], dense[0]) > 1e-3
    assert rel(run(4, (0, 1), bounds_alone), both) < 1e-3


def test_the_last_block_of_the_table_has_positions_of_its_own(cuda):
    """A table of whole blocks holds up to 63 tokens more than max_tokens: each turns by its own angle."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(9)
    layer, n = layer_of(tokens=200), 256
    h = T.randn((n, 512), device="cuda")
    want = plain_attention(layer, h.double().cpu().numpy())
    got = T.cat([layer.attention(h[:190], api.AttnBatch.of([190], [190])), layer.attention(h[190:], api.AttnBatch.of([66], [256]))]).double().cpu().numpy()
    assert rel(got, want) < 0.04 and max(rel(got[i], want[i]) for i in range(n)) < 0.15
