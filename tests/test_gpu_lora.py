"""Low-rank adapters of many tokens beside a shared projection, against the formula in 64 bits.

Tolerance, from the arithmetic: with m = sum_k |A_rk x_k| of a rank's sum and M = |scale| sum_r |B_nr| m_r, z is off by at most u m where u = 2^-16: sums of up to 8192 products in f32 whose
partial sums are rounded (each at most 128 in a row, then a tree or pieces: 160 * 2^-24 < 2^-16) or cut (matrix instructions over operands in parts that hold all their
bits: at most 128 sums in a row, 2^-23 each, beside 2^-20 for what the lesser parts leave); the second product, up to 256 ranks, likewise, and the addition to y rounds once: |error| <= 2^-15 M + 2^-23 (|y| + M).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def check(T, tokens, n_in, n_out, rank, n, act, weights, idx=None, y=True, scale=True, seed=0, lead=0, gap=0, in_place=False, kernel=0):
    from project_maya_b200 import api
    g = T.Generator(device="cuda").manual_seed(seed + tokens + n_in)
    randn = lambda *s: T.randn(s, generator=g, device="cuda")   # noqa: E731
    a, b = (randn(n, rank, n_in) / n_in ** 0.5).to(weights), (randn(n, n_out, rank) / rank ** 0.5).to(weights)
    sc = 0.1 + randn(n).abs() if scale else None
    x = randn(tokens, lead + n_in + gap).to(act)[:, lead:lead + n_in]
    yy = randn(tokens, n_out + gap)[:, :n_out] if y else None
    if idx is None:
        idx = T.randint(-1, n, (tokens,), generator=g, device="cuda", dtype=T.int32)
    ad = api.LoraAdapters(a, b, sc, max_tokens=max(tokens, 32 * n) if kernel == api.LORA_MANY else tokens)
    want, big = (yy.double().clone() if y else T.zeros((tokens, n_out), device="cuda", dtype=T.float64)), T.zeros((tokens, n_out), device="cuda", dtype=T.float64)
    for i in range(n):
        rows = (idx == i).nonzero().flatten()
        if len(rows):
            s = float(sc[i]) if scale else 1.0
            xd, ad64, bd = x[rows].double(), a[i].double(), b[i].double()
            want[rows] += s * (xd @ ad64.T @ bd.T)
            big[rows] = abs(s) * (xd.abs() @ ad64.abs().T @ bd.abs().T)
    base = yy.clone() if y else None
    if in_place:
        out = ad.forward(x, idx, yy, out=yy, kernel=kernel)
        assert out is yy
    else:
        out = ad.forward(x, idx, yy, kernel=kernel)
        assert not y or T.equal(yy, base)
    err = (out.double() - want).abs()
    size = base.double().abs() if y else 0.0
    assert bool((err <= 2.0 ** -15 * big + 2.0 ** -23 * (size + big) + 1e-37).all()), float((err - 2.0 ** -15 * big).max())
    assert ad.error() == 0
    none = (idx < 0) | (idx >= n)
    assert T.equal(out[none], base[none] if y else T.zeros_like(out[none]))
    return ad, x, idx, yy, out


TYPES = [("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"), ("bfloat16", "float16")]


@pytest.mark.parametrize("act,weights", TYPES)
@pytest.mark.parametrize("tokens,n_in,n_out,rank,n", [(1, 32, 1, 1, 1), (1, 4096, 6144, 16, 8), (3, 544, 257, 8, 2), (16, 2048, 1000, 64, 5), (64, 4096, 512, 16, 24),
                                                      (33, 1024, 333, 24, 40), (2, 8192, 130, 256, 3), (100, 512, 96, 100, 7)])
def test_tokens(cuda, act, weights, tokens, n_in, n_out, rank, n):
    import torch as T
    for kernel in (0, 1, 2):
        check(T, tokens, n_in, n_out, rank, n, getattr(T, act), getattr(T, weights), kernel=kernel)


@pytest.mark.parametrize("act,weights", TYPES)
@pytest.mark.parametrize("tokens,n_in,n_out,rank,n", [(200, 1024, 640, 16, 3), (257, 2080, 1001, 64, 2), (1000, 512, 300, 8, 50), (700, 4096, 264, 32, 1),
                                                      (300, 96, 6144, 48, 5), (513, 1024, 200, 128, 4), (300, 1024, 72, 256, 2), (2500, 640, 129, 16, 300)])
def test_prompts(cuda, act, weights, tokens, n_in, n_out, rank, n):
    import torch as T
    for kernel in (0, 2):
        check(T, tokens, n_in, n_out, rank, n, getattr(T, act), getattr(T, weights), kernel=kernel)


@pytest.mark.parametrize("tokens", [1, 40, 300, 900])
def test_who_uses_which(cuda, tokens):
    """Everyone the same, everyone none, numbers outside, runs of requests."""
    import torch as T
    i32 = lambda v: T.tensor(v, dtype=T.int32, device="cuda")   # noqa: E731
    for idx in ([1] * tokens, [-1] * tokens, [(7, -9, 3, 1 << 30)[t % 4] for t in range(tokens)], [t * 5 // tokens - 1 for t in range(tokens)],
                [0] * (tokens - 1) + [3]):
        for kernel in (1, 2):
            check(T, tokens, 512, 320, 16, 4, T.float32, T.bfloat16, idx=i32(idx), kernel=kernel)


@pytest.mark.parametrize("tokens", [5, 300])
def test_without_y_or_scale_in_place_and_rows_apart(cuda, tokens):
    import torch as T
    for n_out in (256, 301):
        for kernel in (1, 2):
            check(T, tokens, 512, n_out, 16, 3, T.float32, T.bfloat16, y=False, kernel=kernel)
            check(T, tokens, 512, n_out, 16, 3, T.float32, T.float16, scale=False, kernel=kernel)
            check(T, tokens, 512, n_out, 80, 3, T.float32, T.bfloat16, in_place=True, kernel=kernel)
            check(T, tokens, 512, n_out, 16, 3, T.bfloat16, T.bfloat16, lead=8, gap=24, kernel=kernel)
            check(T, tokens, 512, n_out, 16, 3, T.float32, T.float16, lead=4, gap=12, in_place=True, kernel=kernel)
            check(T, tokens, 512, n_out, 200, 3, T.float32, T.float16, y=False, kernel=kernel)


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("tokens", [3, 400])
def test_large_and_small_values(cuda, tokens, kernel):
    """Rows of 1e27 beside rows of 1e-27: each token by itself."""
    import torch as T
    from project_maya_b200 import api
    a, b = (T.randn((2, 16, 512), device="cuda") / 22).bfloat16(), (T.randn((2, 256, 16), device="cuda") / 4).bfloat16()
    ad = api.LoraAdapters(a, b, max_tokens=max(tokens, 64))
    x = T.randn((tokens, 512), device="cuda")
    idx = (T.arange(tokens, device="cuda") % 2).int()
    out = ad.forward(x, idx, kernel=kernel)
    up = 2.0 ** ((T.arange(tokens, device="cuda") % 3 - 1) * 90).float()[:, None]
    got = ad.forward(x * up, idx, kernel=kernel)
    assert bool(((got / up - out).abs() <= 2.0 ** -20 * out.abs().amax(1, keepdim=True)).all())
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    bad = ad.forward(x, idx, kernel=kernel)
    assert bool(bad[1].isnan().all()) and not bool(bad[2].isfinite().any())
    keep = [t for t in range(tokens) if t not in (1, 2)]
    assert T.equal(bad[keep], out[keep])


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("tokens", [4, 500])
def test_the_same_call_again_another_stream_and_captured(cuda, tokens, kernel):
    import torch as T
    ad, x, idx, y, out = check(T, tokens, 1024, 520, 32, 6, T.float32, T.bfloat16, kernel=kernel)
    assert T.equal(ad.forward(x, idx, y, kernel=kernel), out)
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(s):
        other = ad.forward(x, idx, y, kernel=kernel)
    s.synchronize()
    assert T.equal(other, out)
    g, got = T.cuda.CUDAGraph(), T.empty_like(out)
    with T.cuda.graph(g, stream=s):
        ad.forward(x, idx, y, out=got, kernel=kernel)
    x2, idx2 = x.flip(0).clone(), idx.flip(0).clone()
    want = ad.forward(x2, idx2, y, kernel=kernel)
    x.copy_(x2)
    idx.copy_(idx2)
    g.replay()
    assert T.equal(got, want)


def test_beside_a_product(cuda):
    """The shared projection (GGUF rows), then the adapters onto its output."""
    import torch as T
    from project_maya_b200 import api
    w = api.synth_weights(api.Q8_0, 1, 0.02, 256, 512)
    for tokens in (1, 8):
        x = T.randn((tokens, 512), device="cuda")
        a, b = (T.randn((3, 16, 512), device="cuda") / 22).half(), (T.randn((3, 256, 16), device="cuda") / 4).half()
        ad, idx = api.LoraAdapters(a, b), T.tensor([t % 4 - 1 for t in range(tokens)], dtype=T.int32, device="cuda")
        y = api.native_mmvq(api.Q8_0, w, api.native_quantize_q8_1(x), 512, 256, tokens)
        delta = ad.forward(x, idx)
        both = ad.forward(x, idx, y)
        assert bool(((both - (y + delta)).abs() <= 2.0 ** -22 * (y.abs() + delta.abs())).all())
        assert T.equal(ad.forward(x, idx, y, out=y), both)


def test_more_tokens_than_the_scratch_is_for(cuda):
    import torch as T
    from project_maya_b200 import api
    ad = api.LoraAdapters(T.zeros((1, 16, 64), device="cuda").half(), T.zeros((1, 64, 16), device="cuda").half(), max_tokens=4)
    with pytest.raises(api.MayaError) as e:
        ad.forward(T.zeros((5, 64), device="cuda"), T.zeros(5, dtype=T.int32, device="cuda"))
    assert e.value.status == -4
    assert ad.forward(T.zeros((0, 64), device="cuda"), T.zeros(0, dtype=T.int32, device="cuda")).shape == (0, 64)


@pytest.mark.parametrize("rank", [16, 80])
def test_calls_in_place_that_nobody_takes_part_in(cuda, rank):
    """Every other call has nothing to do: none of its blocks may be a call ahead of the scratch that they look their tiles up in."""
    import torch as T
    from project_maya_b200 import api
    ad, x, idx, y, out = check(T, 400, 512, 320, rank, 3, T.float32, T.bfloat16, kernel=api.LORA_MANY)
    none, kept = T.full_like(idx, -1), y.clone()
    got = [T.empty_like(out) for _ in range(20)]
    for o in got:
        ad.forward(x, none, y, out=y, kernel=api.LORA_MANY)
        ad.forward(x, idx, y, out=o, kernel=api.LORA_MANY)
    assert all(T.equal(o, out) for o in got) and T.equal(y, kept) and ad.error() == 0


@pytest.mark.parametrize("act,weights", TYPES)
@pytest.mark.parametrize("rank,n_out", [(16, 256), (80, 301)])
@pytest.mark.parametrize("kernel", [1, 2])
def test_infinities_are_those_of_the_formula(cuda, act, weights, rank, n_out, kernel):
    """An infinity stays one until it meets another sign, a zero or a NaN, whichever kernel serves the call.  Whether a sum is infinite or no number does not depend on
    its order (nothing overflows here), so that 64 bits say it.  Adapter 0: positive A, an output's B of one sign; 1: weights of either sign; 2: positive A with zeros; 3:
    scale 0; 4: all positive."""
    import torch as T
    from project_maya_b200 import api
    g = T.Generator(device="cuda").manual_seed(rank)
    n, n_in, tokens = 5, 544, 300
    a, b = T.randn((n, rank, n_in), generator=g, device="cuda") / 16, T.randn((n, n_out, rank), generator=g, device="cuda") / 4
    a[0], a[2] = a[0].abs() + 0.01, a[2].abs() + 0.01
    b[0] = (b[0].abs() + 0.01) * T.where(T.arange(n_out, device="cuda") % 2 == 0, 1.0, -1.0)[:, None]
    a[4], b[4] = a[4].abs() + 0.01, b[4].abs() + 0.01
    a[0, :, ::2] = 0.125                                                           # (in f16: no second term)
    a[2, 3, 7] = b[0, 5, 2] = 0.0
    a, b = a.to(getattr(T, weights)), b.to(getattr(T, weights))
    scale = T.tensor([0.5, 2.0, -1.0, 0.0, 3.0], device="cuda")
    idx = (T.arange(tokens, device="cuda") % 7 - 1).int()                          # (-1 and 5: none)
    clean = T.randn((tokens, n_in), generator=g, device="cuda").to(getattr(T, act))
    x = clean.clone()
    x[20:40, 4] = float("inf")
    x[40:60, 7] = -float("inf")
    x[60:70, 100], x[60:70, 101] = float("inf"), -float("inf")
    x[70:80, 543] = float("nan")
    x[80:100, 300:310] = float("inf")
    y = T.randn((tokens, n_out), generator=g, device="cuda")
    y[100:120, 3], y[20:30, 3] = float("inf"), -float("inf")
    want = y.double()
    for i in range(n):
        rows = idx == i
        want[rows] += float(scale[i]) * (x[rows].double() @ a[i].double().T @ b[i].double().T)
    ad = api.LoraAdapters(a, b, scale, max_tokens=tokens)
    out = ad.forward(x, idx, y, kernel=kernel)
    assert T.equal(out.isnan(), want.isnan())
    assert T.equal(out.isposinf(), want.isposinf()) and T.equal(out.isneginf(), want.isneginf())
    assert bool(want[20:60].isposinf().any()) and bool(want[20:60].isneginf().any())
    same = lambda u, v: T.allclose(u, v, rtol=0.0, atol=0.0, equal_nan=True)       # noqa: E731
    assert same(out[120:], ad.forward(clean, idx, y, kernel=kernel)[120:])
    twice = y.clone()
    assert same(ad.forward(x, idx, twice, out=twice, kernel=kernel), out) and ad.error() == 0


@pytest.mark.parametrize("act,weights", TYPES)
@pytest.mark.parametrize("rank", [16, 64, 80, 256])
@pytest.mark.parametrize("product", ["first", "second"])
@pytest.mark.parametrize("kernel", [1, 2])
def test_operands_keep_their_last_bits(cuda, act, weights, rank, product, kernel):
    """Pairs of terms that differ in their last bits alone, so that the leading parts cancel and only the least are left.  All values are whole numbers times one power of two,
    every product and every sum of any order is one below 2^24: nothing rounds, and the result is equal to the whole numbers'."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(rank)
    n, n_in, tokens = 3, 544, 300
    at = rng.permutation(n_in)
    idx = rng.integers(-1, n, tokens).astype(np.int32)
    x_most, w_most = 24 if act == "float32" else 8, 11 if weights == "float16" else 8
    half = rank // 2
    ranks = rng.permutation(rank)
    pairs = rank if product == "first" else half
    p, q = (at[:rank], at[rank:2 * rank]) if product == "first" else (at[ranks[:half]], at[ranks[half:]])         # where a pair's values lie in x
    whole = lambda bits, shape: rng.integers(1 << (bits - 1), 1 << bits, shape)    # noqa: E731
    other = lambda v, low: (v >> low << low) + rng.integers(0, 1 << low, v.shape)  # noqa: E731
    for x_bits, x_low, w_bits, w_low in ((x_most, x_most // 3, 1, 0), (1, 0, w_most, 3), (min(x_most, 12), 3, w_most, 3)):
        X = np.where(rng.random((tokens, n_in)) < 0.5, 1, -1) * whole(x_bits, (tokens, n_in))
        m, w = whole(x_bits, (tokens, pairs)), whole(w_bits, (n, pairs)) * np.where(rng.random((n, pairs)) < 0.5, 1, -1)
        m2, w2 = other(m, x_low), np.sign(w) * other(abs(w), w_low)
        X[:, p], X[:, q] = m, m2
        A, B = np.zeros((n, rank, n_in), np.int64), np.zeros((n, rank + 3, rank), np.int64)
        out_at = np.arange(pairs)
        if product == "first":
            A[:, out_at, p], A[:, out_at, q] = w, -w2
            B[:, out_at, out_at] = 1
        else:
            A[:, np.arange(rank), at[:rank]] = 1
            B[:, out_at, ranks[:half]], B[:, out_at, ranks[half:]] = w, -w2
        want = np.zeros((tokens, rank + 3))
        has = idx >= 0
        want[has, :pairs] = (w[idx] * m - w2[idx] * m2)[has]
        x, a, b = (T.from_numpy(v.astype(np.float64)).cuda().to(getattr(T, t)) for v, t in ((X * 2.0 ** -9, act), (A, weights), (B, weights)))
        assert T.equal(x.double().cpu(), T.from_numpy(X * 2.0 ** -9)) and np.abs(want).max() < 2.0 ** 24
        for n_out in (rank + 3, rank):
            ad = api.LoraAdapters(a, b[:, :n_out].contiguous(), max_tokens=tokens)
            out = ad.forward(x, T.from_numpy(idx).cuda(), kernel=kernel)
            assert T.equal(out.double().cpu(), T.from_numpy(want[:, :n_out] * 2.0 ** -9))
        assert ad.error() == 0 and bool((want != 0).any())
