"""A decoder layer that serves many requests: adapters beside its products, blocks handed out as they are needed, sequences forked, freed and moved, routing over groups of
experts, norms that leave 8-bit rows - each against the layer without it, and all of them in one run."""
import numpy as np
import pytest

from test_gpu_decoder_layer import plain_attention, rel

pytestmark = pytest.mark.gpu


def layer_of(api, n_seq=1, tokens=400, **more):
    from project_maya_b200 import decoder_layer as L
    norm8 = more.pop("norm_8_bits", False)
    cfg = L.AttentionConfig(512, 8, 2, 64, norm_8_bits=norm8)
    return L.synthetic_layer(cfg, api.MoeLayerConfig(512, 256, 16, 2, api.Q8_0, api.Q8_0), tokens, 512, n_seq=n_seq, **more)


def adapters_of(T, api, n=3, rank=8, rows=768, width=512, seed=3):
    g = T.Generator(device="cuda").manual_seed(seed)
    make = lambda n_in, n_out: api.LoraAdapters((T.randn((n, rank, n_in), generator=g, device="cuda") / n_in ** 0.5).bfloat16(),   # noqa: E731
                                                (T.randn((n, n_out, rank), generator=g, device="cuda") / rank ** 0.5).bfloat16(), 0.5 * T.ones(n, device="cuda"), 512)
    return {"qkv": make(width, rows), "o": make(512, width)}


def test_norms_in_8_bits(cuda):
    """The layer with and without: the same but for sums in another order, which move a code here and there - one in thousands, by a step, 1 % of a value's rms:
    1e-3 (as for attention's sums in another order)."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(1)
    h = T.randn((320, 512), device="cuda")
    a, b = layer_of(api), layer_of(api, norm_8_bits=True)
    at = 0
    for new in (200, 64, 9, 8, 1, 3, 35):
        batch = api.AttnBatch.of([new], [at + new])
        x, y = (layer.attention(h[at:at + new], batch).double().cpu().numpy() for layer in (a, b))
        assert rel(y, x) < 1e-3
        x, y = (layer.forward(h[at:at + new], batch) for layer in (a, b))          # (the same tokens again: their keys stay what they are)
        err = ((x - y).norm(dim=1) / x.norm(dim=1)).cpu().numpy()
        assert np.median(err) < 2e-3 and np.isfinite(err).all()                    # (a token may be routed elsewhere where two scores are near)
        at += new


@pytest.mark.parametrize("norm_8_bits", [False, True])
def test_adapters(cuda, norm_8_bits):
    """Against the attention half in 64 bits over weights with the adapters' products added; within the 4 % of its 8-bit roundings, and no adapter: the layer without."""
    import torch as T
    from project_maya_b200 import api
    import test_gpu_decoder_layer as base
    T.manual_seed(2)
    ads = adapters_of(T, api)
    layer, bare = layer_of(api, adapters=ads, norm_8_bits=norm_8_bits), layer_of(api, norm_8_bits=norm_8_bits)
    h = T.randn((300, 512), device="cuda")
    for which in (1, -1):
        got, at = [], 0
        for new in (230, 9, 7, 1, 53):
            idx = T.full((new,), which, dtype=T.int32, device="cuda")
            got.append(layer.attention(h[at:at + new], api.AttnBatch.of([new], [at + new]), idx))
            at += new
        got = T.cat(got).double().cpu().numpy()
        if which < 0:
            at, want = 0, []
            for new in (230, 9, 7, 1, 53):
                want.append(bare.attention(h[at:at + new], api.AttnBatch.of([new], [at + new])))
                at += new
            assert np.array_equal(got, T.cat(want).double().cpu().numpy())
            continue
        plus = {"qkv": 0.5 * (ads["qkv"].b[which].double() @ ads["qkv"].a[which].double()).cpu().numpy(),
                "o": 0.5 * (ads["o"].b[which].double() @ ads["o"].a[which].double()).cpu().numpy()}
        plain = base.dequantize_q8_0
        try:
            base.dequantize_q8_0 = lambda raw, rows, cols: plain(raw, rows, cols) + plus["qkv" if rows == 768 else "o"]
            want = plain_attention(layer, h.double().cpu().numpy())
        finally:
            base.dequantize_q8_0 = plain
        assert rel(got, want) < 0.04
        assert rel(want, plain_attention(layer, h.double().cpu().numpy())) > 0.1                                      # (the adapters matter)


def test_each_token_has_its_own_adapter(cuda):
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(3)
    ads = adapters_of(T, api)
    h = T.randn((4, 60, 512), device="cuda")
    both, alone = layer_of(api, n_seq=4, adapters=ads), [layer_of(api, n_seq=4, adapters=ads) for _ in range(4)]
    which = [2, -1, 0, 2]
    idx = lambda w, n: T.full((n,), w, dtype=T.int32, device="cuda")   # noqa: E731
    at = 0
    for new in (40, 1, 2, 17):
        lens = [at + new] * 4
        got = both.attention(h[:, at:at + new].reshape(-1, 512), api.AttnBatch.of([new] * 4, lens), T.cat([idx(w, new) for w in which])).view(4, new, 512)
        for s in range(4):
            want = alone[s].attention(h[s, at:at + new], api.AttnBatch.of([new if i == s else 0 for i in range(4)], [at + new if i == s else 0 for i in range(4)]), idx(which[s], new))
            assert rel(got[s].double().cpu().numpy(), want.double().cpu().numpy()) < 2e-3           # (other kernels for other numbers of tokens: sums in other orders)
        at += new


def test_a_run_of_them_together(cuda):
    """Prompts, beams, leavers and newcomers through a layer with everything switched on, beside plain layers that hold each sequence alone."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(4)
    i32 = lambda v: T.tensor(v, dtype=T.int32, device="cuda")   # noqa: E731
    ads, routing = adapters_of(T, api), api.GroupRouting(4, 2, 0.05 * T.randn(16, device="cuda"), w_scale=1.5)
    S = 4
    layer = layer_of(api, n_seq=S, adapters=ads, routing=routing, paged=True, norm_8_bits=True)
    ref = layer_of(api, n_seq=S, adapters=ads)                                     # sequence s in blocks of its own
    lens, which = [0] * S, [0, 1, -1, 2]

    def step(new, adapters=None):
        for s in range(S):
            lens[s] += new[s]
        n = sum(new)
        h = T.randn((n, 512), device="cuda")
        batch = api.AttnBatch.of(new, lens)
        idx = i32([which[s] for s in range(S) for _ in range(new[s])])
        assert rel(layer.attention(h, batch, idx).double().cpu().numpy(), ref.attention(h, batch, idx).double().cpu().numpy()) < 3e-3
        out = layer.forward(h, batch, idx)
        assert out.shape == h.shape and bool(T.isfinite(out).all())

    def take(child, parent, n):                                                    # the same in the plain layer: the blocks copied
        for part in ("k", "v", "k_scale", "v_scale"):
            t = getattr(ref.cache, part)
            t[ref.cache.table[child].long()] = t[ref.cache.table[parent].long()].clone()
        lens[child], which[child] = n, which[parent]

    step([100, 65, 0, 0])
    step([1, 1, 0, 0])
    layer.pages.fork(i32([0, 1]), i32([2, 3]), i32([101, 64]))
    take(2, 0, 101)
    take(3, 1, 64)
    for _ in range(30):
        step([1, 1, 1, 1])
    step([3, 4, 2, 1])
    layer.pages.free(i32([1]))
    lens[1], which[1] = 0, 1
    layer.pages.compact()
    assert layer.pages.live.item() == int((layer.pages.refs > 0).sum()) and bool((layer.pages.refs[layer.pages.live.item():] == 0).all())
    step([1, 0, 1, 1])
    step([0, 150, 0, 0])
    step([1, 1, 1, 1])
    assert layer.pages.error() == 0 and layer.attn.error() == 0 and layer.token.error() == 0 and layer.chunk.error() == 0 and ads["qkv"].error() == 0
    held = layer.cache.table[layer.cache.table >= 0]
    assert T.equal(T.bincount(held.long(), minlength=layer.cache.n_blocks).int(), layer.pages.refs)
