"""Attention over the 8-bit cache, its append and its selection where they can go wrong: numbers that are not finite, very large and very small ones,
bounds of the arguments, long contexts.  Helpers and plain forms are those of test_gpu_attention.py, and so are the tolerances where nothing else is said."""
import numpy as np
import pytest

from test_gpu_attention import BLOCK, attend, check, make_cache, plain_attention, plain_rows, plain_select, unpack

pytestmark = pytest.mark.gpu


FORMS = [
    # new tokens, lengths, key/value heads, group, head size, bf16, lists
    ([1, 1, 4], [3000, 70, 2], 2, 4, 128, False, 0),     # tokens; two rows before their sequence
    ([1, 1, 4], [3000, 70, 2], 2, 4, 128, True, 0),
    ([9, 3], [400, 90], 1, 6, 64, False, 0),             # windows
    ([2], [100], 1, 16, 256, True, 0),
    ([150, 40], [150, 20], 2, 2, 128, True, 0),          # prompts, whole; twenty tokens before their sequence
    ([300], [500], 1, 1, 64, True, 0),
    ([50, 50], [7000, 40], 2, 3, 128, True, 0),          # cut into pieces and joined
    ([90], [200], 1, 2, 128, False, 0),                  # in f32
    ([1, 2], [1500, 90], 2, 8, 128, True, 5),            # lists
    ([1800], [1900], 4, 2, 64, True, 4),                 # a warp a list
]


@pytest.mark.parametrize("case", range(len(FORMS)))
def test_queries_that_are_not_finite(cuda, case):
    """One NaN or infinity in a query: that row alone is not finite, in the output and in lse, whichever kernel has it; a row that sees nothing is 0 all the
    same; every other row keeps its bits."""
    import torch as T
    new, lens, n_kv, group, dim, bf16, n_sel = FORMS[case]
    rng = np.random.default_rng(600 + case)
    cache, _ = make_cache(T, rng, lens, n_kv, dim)
    N, H = sum(new), n_kv * group
    q = T.from_numpy(rng.standard_normal((N, H, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32).cuda()
    sel = None
    if n_sel:
        own = np.concatenate([(n - m + np.arange(m)) // BLOCK for m, n in zip(new, lens)])
        sel = T.from_numpy(np.sort(np.where(np.arange(n_sel) <= own[:, None, None], own[:, None, None] - np.arange(n_sel), -1).repeat(n_kv, 1).astype(np.int32), -1)).cuda()
    pos = np.concatenate([n - m + np.arange(m) for m, n in zip(new, lens)])
    bad = T.zeros((N, H), dtype=T.bool, device="cuda")
    clean = q.clone()
    for i, x in enumerate((float("nan"), float("inf"), -float("inf"))):
        for row in (i * 7 % N, N - 1 - i * 5 % N):
            bad[row, i % H] = True
            q[row, i % H, (11 * i + 3) % dim] = x
            clean[row, i % H] = 0
    out, lse = attend(T, cache, new, lens, q, sel=sel)
    want, want_lse = attend(T, cache, new, lens, clean, sel=sel)
    seen = T.from_numpy(pos >= 0).cuda()
    lost = bad & seen[:, None]
    assert lost.any() and not T.isfinite(out[lost]).any() and T.isnan(lse[lost]).all()
    assert (out[~seen] == 0).all() and T.isneginf(lse[~seen]).all()
    assert T.equal(out[~lost], want[~lost]) and T.equal(lse[~lost], want_lse[~lost])


@pytest.mark.parametrize("bf16,new,length", [(False, 3, 300), (True, 3, 300), (True, 140, 300)])
def test_queries_of_any_finite_size(cuda, bf16, new, length):
    """Rows near the largest and the smallest normal number, with a scale that brings their scores back."""
    import torch as T
    rng = np.random.default_rng(61)
    cache, host = make_cache(T, rng, [length], 1, 64)
    x = rng.standard_normal((new, 1, 64))
    for size, scale in ((2.0 ** 126 / np.abs(x).max(), 0.125 * 2.0 ** -123), (2.0 ** -124 / np.abs(x).max(), 0.125 * 2.0 ** 122)):
        q = T.from_numpy((x * size).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
        want = plain_attention(host, [new], [length], q.double().numpy(), 1, float(np.float32(scale)))
        out, lse = attend(T, cache, [new], [length], q.cuda(), scale=scale)
        check(out, lse, want, bf16)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 70, 40000])
@pytest.mark.parametrize("new,length,group,bf16", [(1, 30000, 1, False), (4, 30000, 2, True), (5, 3, 1, False), (140, 9000, 1, True), (200, 130, 1, True)])
def test_windows_wider_than_the_context(cuda, window, new, length, group, bf16):
    """The same as no window, up to the largest number there is."""
    import torch as T
    rng = np.random.default_rng(62)
    cache, _ = make_cache(T, rng, [length], 1, 64)
    q = T.from_numpy(rng.standard_normal((new, group, 64)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32).cuda()
    want, want_lse = attend(T, cache, [new], [length], q)
    out, lse = attend(T, cache, [new], [length], q, window=window)
    assert T.equal(out, want) and T.equal(lse, want_lse)


LONG = [
    # new tokens, tokens, group, head size, selected, first, last
    (1, 1 << 20, 1, 64, 40, 1, 1),               # the longest context that the header names, for every size of group: one list by a whole thread block
    (1, 1 << 20, 2, 64, 7, 0, 1),
    (2, (1 << 20) - 30, 4, 64, 16, 1, 2),        # a warp a list
    (1, 1 << 20, 8, 64, 512, 2, 3),
    (3, 1 << 20, 1, 64, 33, 0, 2),
    (2, 300000, 16, 128, 20, 1, 2),
    (30, 40000, 8, 128, 16, 1, 2),
    (40, 70001, 3, 64, 100, 1, 1),
    (9, 140000, 40, 64, 12, 1, 1),
]


@pytest.mark.parametrize("case", range(len(LONG)))
def test_select_over_long_contexts(cuda, case):
    """Lists over more blocks than a warp's (256) or a thread block's (2048) registers hold, up to 16384 blocks; many places share a block of the cache."""
    import torch as T
    from project_maya_b200 import api
    new, n, group, dim, n_sel, n_first, n_last = LONG[case]
    rng = np.random.default_rng(630 + case)
    cache, host = make_cache(T, rng, [90 * BLOCK], 1, dim)
    host["table"] = rng.integers(0, cache.n_blocks, (1, -(-n // BLOCK))).astype(np.int32)
    cache = api.KvCache(cache.k, cache.v, cache.k_scale, cache.v_scale, T.from_numpy(host["table"]).cuda(), cache.k_sum)
    q = T.from_numpy(rng.standard_normal((new, group, dim)).astype(np.float32))
    attn = api.KvAttention(cache, group, n_sel=n_sel, n_first=n_first, n_last=n_last)
    sel = attn.select(api.AttnBatch.of([new], [n]), q.cuda(), sel=T.full((new, 1, n_sel), -5, dtype=T.int32, device="cuda"))
    assert np.array_equal(sel.cpu().numpy(), plain_select(host, [new], [n], q.numpy(), 1, n_sel, n_first, n_last))


def test_select_beyond_the_longest_context_is_refused(cuda):
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(64)
    cache, _ = make_cache(T, rng, [90], 1, 64, wide=16385)
    q = T.zeros((1, 1, 64), device="cuda")
    with pytest.raises(api.MayaError) as e:
        api.KvAttention(cache, 1, n_sel=4).select(api.AttnBatch.of([1], [(1 << 20) + 1]), q)
    assert e.value.status == -4


@pytest.mark.parametrize("new,n,group", [(1, 5000, 4), (20, 5000, 1), (1, 5000, 12)])
def test_select_passes_over_blocks_the_table_does_not_have(cuda, new, n, group):
    """Keys that all point away from the queries: every real block scores below 0, and still stands before one that is not there."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(65)
    cache, host = make_cache(T, rng, [n], 1, 64)
    q = T.from_numpy(rng.uniform(0.5, 1, (new, group, 64)).astype(np.float32))
    host["sums"][:] = rng.integers(-4000, -1000, host["sums"].shape)
    cache.k_sum.copy_(T.from_numpy(host["sums"]))
    gone = rng.permutation(np.arange(1, n // BLOCK - 5))[:30]
    cache.table[0, T.from_numpy(gone).cuda()] = T.from_numpy(np.where(np.arange(30) % 2, -1, cache.n_blocks).astype(np.int32)).cuda()
    attn, batch = api.KvAttention(cache, group, n_sel=12, n_first=1, n_last=2), api.AttnBatch.of([new], [n])
    sel = attn.select(batch, q.cuda()).cpu().numpy()
    assert not np.isin(sel, gone).any() and (sel >= 0).all()
    # the same list as with scores below every real one in their places
    host["ks"][host["table"][0, gone]] = 1e6
    assert np.array_equal(sel, plain_select(host, [new], [n], q.numpy(), 1, 12, 1, 2))
    # fewer real ones than entries: they are all there
    few = api.KvAttention(cache, group, n_sel=60, n_first=1, n_last=2).select(batch, q.cuda()).cpu().numpy()
    real = np.setdiff1d(np.arange((n - new) // BLOCK + 1), gone)
    assert all(np.isin(real, few[i]).all() for i in range(new))


@pytest.mark.parametrize("size", [1e-36, 3e-37, 1e-38, 1e-40, 1e-44])
def test_append_of_the_smallest_values(cuda, size):
    """Values whose 127th is no normal number: a scale is 2^-126 at least, and a code is off by half of it at most."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(66)
    for new, dim in ((1, 64), (40, 128)):
        cache = api.KvCache.empty(1, 1, dim, T.zeros((1, 1), dtype=T.int32, device="cuda"))
        x = (size * rng.uniform(-1, 1, (new, 1, dim))).astype(np.float32)
        d = T.from_numpy(x).cuda()
        api.KvAttention(cache, 1).append(api.AttnBatch.of([new], [new]), d, d, d, api.Rope())
        k, v = unpack(cache)
        for codes, scale in ((k, cache.k_scale), (v, cache.v_scale)):
            s = float(scale.double()[0, 0])
            assert s == max(2.0 ** -126, float(np.float32(np.abs(x).max()) * np.float32(1 / 127)))
            assert (np.abs(codes[0, 0, :new] * s - x[:, 0].astype(np.float64)) <= s * (0.5 + 2.0 ** -15)).all()
        assert np.array_equal(cache.k_sum[0, 0].cpu().numpy(), k[0, 0, :new].sum(0))
        zero = api.KvCache.empty(1, 1, dim, T.zeros((1, 1), dtype=T.int32, device="cuda"))
        api.KvAttention(zero, 1).append(api.AttnBatch.of([new], [new]), d, 0 * d, 0 * d, api.Rope())
        assert float(zero.v_scale) == 0 and (unpack(zero)[1][0, 0, :new] == 0).all()


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("bf16,seqs,new,length", [(False, 1, 1, 4 * BLOCK), (False, 300, 1, 40 * BLOCK), (False, 300, 20, 40 * BLOCK), (True, 300, 1, 40 * BLOCK), (True, 1, 130, 40 * BLOCK)])
def test_value_scales_far_apart(cuda, bf16, seqs, new, length, order):
    """Rows whose weight lies on blocks of small values, beside blocks of values up to 1e15 times as large that they hardly see: off by what P's bits (22 or 11) and
    the scores' error make of sum p |v|, and by what f16 drops of a P 2^-36 (f32; 2^-28 in bf16) of the largest p * value scale - not by a part of the largest value."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(67)
    cache, host = make_cache(T, rng, [length], 1, 64)
    x = rng.standard_normal((1, 1, 64)).repeat(seqs * new, 0)
    x *= rng.uniform(0.9, 1.1, (seqs * new, 1, 1))
    q = T.from_numpy(x.astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    x = q.double().numpy()
    blocks = host["table"][0, :length // BLOCK]
    toward = np.where(x[0, 0] > 0, 1, -1)
    lift = np.linspace(0, 1, len(blocks))[::order]                            # scores from 0 to 60, value scales from 1 down to 1e-15
    for b, f in zip(blocks, lift):
        host["k"][b, 0] = 128 + np.round(toward * rng.uniform(60, 127, (BLOCK, 64)))
        host["ks"][b] = 60 * f / (0.125 * np.abs(x[0, 0]).sum() * 94)
        host["vs"][b] = 10.0 ** (-15 * f)
    raw = host["k"].reshape(*host["k"].shape[:3], 1, 64).transpose(0, 1, 3, 2, 4)
    cache.k.copy_(T.from_numpy(np.ascontiguousarray(raw).astype(np.uint8)))
    cache.k_scale.copy_(T.from_numpy(host["ks"]))
    cache.v_scale.copy_(T.from_numpy(host["vs"]))
    cache = api.KvCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.table.repeat(seqs, 1), cache.k_sum)      # (every sequence reads the same blocks)
    out, lse = attend(T, cache, [new] * seqs, [length] * seqs, q.cuda())
    vs = host["vs"][blocks].astype(np.float64).repeat(BLOCK)
    k = ((host["k"][blocks, 0] - 128) * host["ks"][blocks].astype(np.float64)[..., None]).reshape(-1, 64)
    v = ((host["v"][blocks, 0] - 128) * host["vs"][blocks].astype(np.float64)[..., None]).reshape(-1, 64)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for i in range(0, seqs * new, 1 + seqs * new // 100):
        n = length - new + i % new + 1
        z = 0.125 * (k[:n] @ x[i, 0])
        p = np.exp(z - z.max())
        ref_lse = z.max() + np.log(p.sum())
        p /= p.sum()
        want, A = p @ v[:n], 0.125 * (np.abs(k[:n]) @ np.abs(x[i, 0])).max()
        tol = (2 * 2.0 ** -20 * A + 2.0 ** -19 + (2.0 ** -11 if bf16 else 0)) * (p @ np.abs(v[:n]))
        tol = tol + (2.0 ** -28 if bf16 else 2.0 ** -36) * (p * vs[:n]).max() * 127 * n + (2.0 ** -8 * np.abs(want) if bf16 else 0)
        assert (np.abs(got[i, 0] - want) <= tol).all(), (i, (np.abs(got[i, 0] - want) / tol).max())
        assert abs(got_lse[i, 0] - ref_lse) <= 2 * 2.0 ** -20 * A + 2.0 ** -19 + 2.0 ** -22 * abs(ref_lse)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("new,lens,pairs", [([1, 1], [30, 70], False), ([9, 70], [9, 200], True)])
def test_append_with_positions_of_its_own(cuda, new, lens, pairs, bf16):
    """Rows of cos and sin by `pos`, in any order; those outside the table take the nearest."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(68)
    N, H, n_kv, dim = sum(new), 4, 2, 128
    cache, _ = make_cache(T, rng, lens, n_kv, dim)
    pos = rng.permutation(300)[:N].astype(np.int32) - 40
    pos[0], pos[-1] = 10 ** 9, -10 ** 9
    angle = np.arange(200)[:, None] * 100.0 ** (-np.arange(32) / 32)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    q, k, v = (T.from_numpy(rng.standard_normal((N, heads, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32) for heads in (H, n_kv, n_kv))
    got = api.KvAttention(cache, H).append(api.AttnBatch.of(new, lens), q.cuda(), k.cuda(), v.cuda(), api.Rope(T.from_numpy(cos).cuda(), T.from_numpy(sin).cuda(), pairs=pairs),
                                           pos=T.from_numpy(pos).cuda()).double().cpu().numpy()
    turn = np.clip(pos, 0, 199)
    want = plain_rows(q.double().numpy(), None, cos, sin, turn, 0, pairs)
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want).max(-1, keepdims=True) + (2.0 ** -8 * np.abs(want) if bf16 else 0)).all()
    keys = plain_rows(k.double().numpy(), None, cos, sin, turn, 0, pairs)
    codes, scale = unpack(cache)[0], cache.k_scale.double().cpu().numpy()
    table, row = cache.table.cpu().numpy(), 0
    for s, (m, n) in enumerate(zip(new, lens)):
        for i in range(m):
            at = n - m + i
            b = table[s, at // BLOCK]
            assert (np.abs(codes[b, :, at % BLOCK] * scale[b][:, None] - keys[row + i]) <= scale[b][:, None] * (0.5 + 127 * 2.0 ** -19)).all()
        row += m


@pytest.mark.parametrize("bf16", [False, True])
def test_append_of_queries_alone_and_in_place(cuda, bf16):
    """Without keys and values the cache keeps every byte; queries may be turned where they lie."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(69)
    for new, lens in (([3, 1], [40, 130]), ([200, 9], [200, 70])):
        cache, _ = make_cache(T, rng, lens, 2, 64)
        N, H = sum(new), 6
        held = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_sum)]
        q = T.from_numpy(rng.standard_normal((N, H, 64)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32).cuda()
        angle = T.arange(300, device="cuda")[:, None] * 100.0 ** (-T.arange(32, device="cuda") / 32)
        rope = api.Rope(angle.cos(), angle.sin(), q_w=T.rand(64, device="cuda"))
        attn, batch = api.KvAttention(cache, H), api.AttnBatch.of(new, lens)
        out = attn.append(batch, q, None, None, rope)
        assert attn.append(batch, q, None, None, rope, q_out=q) is q and T.equal(q, out)
        assert all(T.equal(a, b) for a, b in zip(held, (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_sum)))


def test_calls_after_an_error_are_sound(cuda):
    """The error word and counters as a launch that gave up would leave them (set here by the host)."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(70)
    cache, _ = make_cache(T, rng, [20000], 1, 64)
    q, attn, batch = T.randn((1, 2, 64), device="cuda"), api.KvAttention(cache, 2), api.AttnBatch.of([1], [20000])
    want = attn.forward(batch, q)
    attn.scratch[:32].view(T.int32).copy_(T.tensor([1, 0, 0, 0, 3, 5, 0, 0]))
    assert attn.error() == 1 and attn.error() == 0
    assert T.equal(attn.forward(batch, q), want) and attn.error() == 0
