"""Routing over groups of experts against its definition in 64 bits, and the layers that use it.

The choice is made in 64 bits on both sides: ids are equal.  A weight is rounded once to f32 (2^-24) behind 64-bit arithmetic (exp within an ulp, sums
of up to 2048 values: 2^-40 at most): 2^-23 of it.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(logits, k, n_group=1, n_keep=1, bias=None, sigmoid=True, top2=True, norm_w=True, w_scale=1.0):
    T, E = logits.shape
    l = logits.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            s = 1 / (1 + np.exp(-l))
        else:
            top = l.max(1, keepdims=True)
            e = np.exp(l - top)
            s = e / e.sum(1, keepdims=True)
            s[(l == -np.inf).all(1)] = 0.0
        c = s if bias is None else s + bias.astype(np.float64)
    ids, w = np.zeros((T, k), np.int32), np.zeros((T, k))
    # numbers first, from the highest; then what is no number; equal ones by their place
    ranked = lambda v, at: sorted(at, key=lambda i: (np.isnan(v[i]), 0.0 if np.isnan(v[i]) else -v[i], i))   # noqa: E731
    for t in range(T):
        size, seen = E // n_group, range(E)
        if n_keep < n_group:
            score = []
            for g in range(n_group):
                best = [c[t, i] for i in ranked(c[t], range(g * size, (g + 1) * size))]
                with np.errstate(invalid="ignore"):
                    score.append(best[0] + best[1] if top2 and size > 1 else best[0])
            kept = ranked(np.array(score), range(n_group))[:n_keep]
            seen = [i for i in range(E) if i // size in kept]
        ids[t] = ranked(c[t], seen)[:k]
        w[t] = s[t, ids[t]]
        if norm_w:
            total = w[t].sum()
            w[t] /= total if total > 2.0 ** -14 or np.isnan(total) else 2.0 ** -14
    return ids, w * w_scale


def check(T, logits, k, **how):
    from project_maya_b200 import api
    bias = how.get("bias")
    ids, w = api.router_groups(T.from_numpy(logits).cuda(), k, **{**how, "bias": None if bias is None else T.from_numpy(bias).cuda()})
    want_ids, want = plain(logits, k, **how)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(got - want)[ok] <= 2.0 ** -23 * np.abs(want)[ok] + 1e-44).all()


SHAPES = [(1, 256, 8, 8, 4), (61, 160, 6, 8, 3), (300, 256, 8, 8, 4), (5, 2048, 64, 32, 20), (3, 40, 7, 5, 2), (9, 33, 3, 1, 1), (4, 32, 5, 32, 7),
          (2, 7, 7, 7, 7), (1, 1, 1, 1, 1), (150, 512, 10, 2, 1), (7, 1000, 33, 25, 24), (3, 96, 4, 3, 2), (2, 320, 40, 20, 3), (160, 1024, 12, 16, 5)]


@pytest.mark.parametrize("tokens,experts,k,groups,keep", SHAPES)
@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("top2", [True, False])
def test_choice_and_weights(cuda, tokens, experts, k, groups, keep, sigmoid, top2):
    import torch as T
    rng = np.random.default_rng(tokens * experts)
    logits = (2 * rng.standard_normal((tokens, experts))).astype(np.float32)
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    for b, norm_w, w_scale in ((bias, True, 2.5), (None, False, 1.0)):
        check(T, logits, k, n_group=groups, n_keep=keep, bias=b, sigmoid=sigmoid, top2=top2, norm_w=norm_w, w_scale=w_scale)


@pytest.mark.parametrize("sigmoid", [True, False])
def test_equal_scores_go_to_the_lower_expert_and_group(cuda, sigmoid):
    import torch as T
    rng = np.random.default_rng(3)
    logits = rng.integers(-2, 3, (200, 64)).astype(np.float32)
    logits[0] = 0.0
    logits[1, :] = 50.0                                          # sigmoid: all 1
    for top2 in (True, False):
        check(T, logits, 9, n_group=8, n_keep=3, sigmoid=sigmoid, top2=top2)
    check(T, logits, 9, sigmoid=sigmoid, bias=np.zeros(64, np.float32))


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("keep", [2, 8])
def test_rows_with_masked_experts_infinities_and_nan(cuda, sigmoid, keep):
    import torch as T
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((12, 64)).astype(np.float32)
    logits[0] = -np.inf
    logits[1, 3:] = -np.inf
    logits[2] = np.finfo(np.float32).min
    logits[3, 5] = np.nan
    logits[4] = np.nan
    logits[5, 60] = np.inf
    logits[6, 8:16] = np.nan
    logits[7, :63] = -np.inf
    logits[7, 63] = np.nan
    logits[8] = np.finfo(np.float32).max
    logits[9, ::2] = -1e4
    for top2 in (True, False):
        check(T, logits, 6, n_group=8, n_keep=keep, sigmoid=sigmoid, top2=top2)
    bias = np.zeros(64, np.float32)
    bias[10:40] = -np.inf
    check(T, logits, 6, n_group=8, n_keep=keep, sigmoid=sigmoid, bias=bias)


def test_neighbours_that_f32_cannot_tell_apart(cuda):
    """Saturated sigmoids: 1 - 1e-9 and less apart, equal in f32 and ordered in f64."""
    import torch as T
    rng = np.random.default_rng(5)
    logits = rng.uniform(18, 30, (64, 128)).astype(np.float32)
    check(T, logits, 8, n_group=4, n_keep=2)
    check(T, logits, 8)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("spread", [0.01, 1.5, 40.0])
def test_many_tokens(cuda, sigmoid, spread):
    """Tens of thousands of borders, among them all degrees of nearness, with and without a bias."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(int(spread * 100))
    logits, bias = spread * T.randn((20000, 256), device="cuda"), 0.05 * T.randn(256, device="cuda")
    for b in (bias, None):
        s = T.sigmoid(logits.double()) if sigmoid else T.softmax(logits.double(), -1)
        c = s if b is None else s + b.double()
        groups = c.view(-1, 8, 32).sort(dim=-1, descending=True).values[..., :2].sum(-1).sort(dim=-1, descending=True, stable=True).indices[:, :4]
        seen = T.zeros((20000, 8), dtype=T.bool, device="cuda").scatter_(1, groups, True).repeat_interleave(32, 1)
        want = c.masked_fill(~seen, -float("inf")).sort(dim=-1, descending=True, stable=True).indices[:, :8]
        ids, w = api.router_groups(logits, 8, 8, 4, b, sigmoid)
        assert T.equal(ids.long(), want)
        p = s.gather(1, want)
        p = p / p.sum(-1, keepdim=True).clamp(min=2.0 ** -14)
        assert bool(((w.double() - p).abs() <= 2.0 ** -23 * p + 1e-44).all())


def test_the_same_beside_others_and_captured(cuda):
    import torch as T
    from project_maya_b200 import api
    logits = T.randn((500, 256), device="cuda")
    how = dict(n_group=8, n_keep=4, bias=0.1 * T.randn(256, device="cuda"))
    ids, w = api.router_groups(logits, 8, **how)
    for t in (0, 3, 499):
        i1, w1 = api.router_groups(logits[t:t + 1], 8, **how)
        assert T.equal(i1[0], ids[t]) and T.equal(w1[0], w[t])
    out = T.empty_like(ids), T.empty_like(w)
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        api.router_groups(logits, 8, ids=out[0], weights=out[1], **how)
    logits.copy_(logits.flip(0))
    g.replay()
    assert T.equal(out[0], ids.flip(0)) and T.equal(out[1], w.flip(0))


def layer_config(api, gu_type=None):
    return api.MoeLayerConfig(512, 256, 32, 4, gu_type or api.Q4_K, api.Q8_0)


def experts_of(T, api, cfg):
    blobs = T.empty((cfg.n_expert, cfg.blob_bytes), dtype=T.uint8, device="cuda")
    gu = 2 * cfg.n_ff * api.row_bytes(cfg.gu_type, cfg.n_embd)
    for e in range(cfg.n_expert):
        api.synth_weights(cfg.gu_type, e + 1, 0.05, 2 * cfg.n_ff, cfg.n_embd, blobs[e, :gu])
        api.synth_weights(cfg.d_type, e + 101, 0.05, cfg.n_embd, cfg.n_ff, blobs[e, gu:])
    return blobs


def test_routed_layer_equals_the_layer_that_routes(cuda):
    """Tokens routed by router_top10 and handed over: the staged layer's bits."""
    import torch as T
    from project_maya_b200 import api
    cfg = layer_config(api)
    blobs = experts_of(T, api, cfg)
    layer = api.MoeLayer(cfg, blobs, staged=True)
    for n in (1, 2, 7, 16):
        for dt in (T.float32, T.bfloat16):
            logits, x = T.randn((n, 32), device="cuda"), T.randn((n, 512), device="cuda").to(dt)
            ids, w, out = layer.forward(logits, x)
            assert T.equal(layer.forward_routed(ids, w, x), out)
    assert layer.error() == 0


def test_routed_layer_leaves_out_ids_that_are_none(cuda):
    import torch as T
    from project_maya_b200 import api
    cfg = layer_config(api)
    layer = api.MoeLayer(cfg, experts_of(T, api, cfg), staged=True)
    x = T.randn((3, 512), device="cuda")
    ids = T.tensor([[1, -1, 5, 40], [-1, -7, 32, 1 << 30], [2, 3, 4, 5]], dtype=T.int32, device="cuda")
    w = T.rand((3, 4), device="cuda")
    out = layer.forward_routed(ids, w, x)
    some = T.tensor([[1, 5, 1, 5], [0, 1, 2, 3], [2, 3, 4, 5]], dtype=T.int32, device="cuda")
    part = w[:, [0, 2, 1, 3]].clone()
    part[0, 2:] = 0.0
    part[1] = 0.0
    part[2] = w[2]
    want = layer.forward_routed(some, part, x)
    assert bool((out[1] == 0).all())
    assert T.allclose(out, want, rtol=1e-5, atol=1e-6 * float(want.abs().max()))       # (terms of 0 among the sums)
    assert layer.error() == 0


def test_layers_with_group_routing(cuda):
    """Windows and prompts route as router_groups does, and agree.  Both round x and h to 8 bits; the prompt path keeps the products scale * code in f16 (2^-11), which
    moves an h by up to an eighth of its step (127 steps * 2^-10) and so one code in sixteen by a step, 1/40 of the values' rms: 0.6 % beside 0.2 %.  Below 2 %."""
    import torch as T
    from project_maya_b200 import api
    cfg = layer_config(api, api.Q8_0)
    blobs = experts_of(T, api, cfg)
    routing = api.GroupRouting(4, 2, 0.1 * T.randn(32, device="cuda"), w_scale=2.5)
    token, chunk = api.MoeLayer(cfg, blobs, routing=routing), api.MoePrefill(cfg, blobs, max_tokens=64, routing=routing)
    logits, x = T.randn((40, 32), device="cuda"), T.randn((40, 512), device="cuda")
    want_ids, want_w = api.router_groups(logits, 4, 4, 2, routing.bias, w_scale=2.5)
    ids, w, ffn = (v.clone() for v in chunk.forward(logits, x))
    assert T.equal(ids, want_ids) and T.equal(w, want_w)
    for a, b in ((0, 16), (16, 17), (17, 30)):
        i1, w1, out = token.forward(logits[a:b], x[a:b])
        assert T.equal(i1, want_ids[a:b]) and T.equal(w1, want_w[a:b])
        assert float((out - ffn[a:b]).norm() / out.norm()) < 2e-2
    assert token.error() == 0 and chunk.error() == 0
    with pytest.raises(api.MayaError):
        token.forward_checked(logits[:1], x[:1], api.LAYER_STAGED)
    with pytest.raises(api.MayaError):
        token.forward(logits[:1], x[:1], hc=(x, x, x, x))


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("large", [64.0, 1e2, 1e3, 1e5, 1e6])
@pytest.mark.parametrize("where", ["every group", "one group"])
def test_large_biases_that_cancel_in_a_group(cuda, sigmoid, large, where):
    """A pinned expert beside a banned one: the group's sum is small and the rounding of the two is not, 2^-24 of each bias in 32 bits.  In every group the borders
    themselves are in doubt; in one, a group that stands away from the border may belong on its other side."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(int(large))
    logits = (0.01 if where == "every group" else 0.5) * T.randn((100000, 16), device="cuda")
    bias = T.zeros(16, device="cuda")
    pairs = bias.view(8, 2)[:8 if where == "every group" else 1]
    pairs[:, 0], pairs[:, 1] = large, -large
    s = T.sigmoid(logits.double()) if sigmoid else T.softmax(logits.double(), -1)
    c = s + bias.double()
    groups = c.view(-1, 8, 2).sort(dim=-1, descending=True).values.sum(-1).sort(dim=-1, descending=True, stable=True).indices[:, :4]
    seen = T.zeros((100000, 8), dtype=T.bool, device="cuda").scatter_(1, groups, True).repeat_interleave(2, 1)
    want = c.masked_fill(~seen, -float("inf")).sort(dim=-1, descending=True, stable=True).indices[:, :3]
    ids, w = api.router_groups(logits, 3, 8, 4, bias, sigmoid)
    assert T.equal(ids.long(), want)
    p = s.gather(1, want)
    assert bool(((w.double() - p / p.sum(-1, keepdim=True)).abs() <= 2.0 ** -23).all())


def test_routed_layer_takes_nothing_from_the_weights_of_ids_that_are_none(cuda):
    """Whatever stands in a masked place - an infinity, NaN - the output is that of a weight of 0 there; an id given twice counts twice."""
    import torch as T
    from project_maya_b200 import api
    cfg = layer_config(api)
    blobs = experts_of(T, api, cfg)
    x, w = T.randn((5, 512), device="cuda"), T.rand((5, 4), device="cuda")
    ids = T.tensor([[1, -1, 5, 40], [-1, -7, 32, 1 << 30], [2, 3, 4, -1], [6, 6, 6, 6], [7, 1, 7, -1]], dtype=T.int32, device="cuda")
    none = (ids < 0) | (ids >= 32)
    for layer in (api.MoeLayer(cfg, blobs, staged=True), api.MoeLayer(cfg, blobs, expert_range=(0, 5))):
        want = layer.forward_routed(ids, w.masked_fill(none, 0.0), x)
        assert bool(want.isfinite().all()) and bool((want[1] == 0).all())
        for odd in (float("nan"), float("inf"), -float("inf"), 3e38):
            assert T.equal(layer.forward_routed(ids, w.masked_fill(none, odd), x), want)
        assert layer.error() == 0
    once = T.tensor([[6, -1, -1, -1]], dtype=T.int32, device="cuda")
    layer = api.MoeLayer(cfg, blobs, staged=True)
    four, one = layer.forward_routed(ids[3:4], w[3:4], x[3:4]), layer.forward_routed(once, T.stack([w[3].sum()] + [w[3, 0]] * 3)[None], x[3:4])
    assert bool(((four - one).abs() <= 2.0 ** -21 * w[3].sum() * (one / w[3].sum()).abs()).all())        # (four products and sums of one sign, each rounded: 8 * 2^-24)


@pytest.mark.parametrize("top2", [True, False])
@pytest.mark.parametrize("keep,k", [(3, 30), (3, 31), (2, 20), (1, 10)])
def test_choices_that_run_out_of_numbers(cuda, top2, keep, k):
    """Fewer scores that are numbers than choices: NaN are chosen, and a sum with one is none, so no weight of a normalised token is a number."""
    import torch as T
    rng = np.random.default_rng(10 * keep + k)
    logits = rng.standard_normal((20, 42)).astype(np.float32)
    logits[:, ::4] = np.nan
    logits[4, ::2] = np.nan
    logits[7] = 0.5
    for w_scale in (1.0, -1.0):
        for norm_w in (True, False):
            check(T, logits, k, n_group=3, n_keep=keep, norm_w=norm_w, top2=top2, w_scale=w_scale)
