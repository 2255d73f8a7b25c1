"""Attention over the paged 8-bit cache, the append in front of it and the block selection, against plain implementations in 64 bits.

Tolerances, from the arithmetic (not from a run): with A = scale * sum |q_d k_d| of a score and vmax = max |v| of the rows it sees,
  f32:  q and P are two f16 terms (22 bits), sums are f32: a score is off by at most 2^-20 A (and 2^-22 from the exponential), so the
        output by 2 * 2^-20 A vmax + 2^-19 vmax
  bf16: q is exact in f16, P is rounded to 11 bits: 2^-11 vmax beside the f32 terms, and the result's own rounding, 2^-8 |out|.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BLOCK = 64


def make_cache(T, rng, lens, n_kv, dim, spare=5, wide=None):
    """A cache with random codes and scales for sequences of `lens` tokens, its blocks in random order; unused entries -1."""
    from project_maya_b200 import api
    need = [-(-n // BLOCK) for n in lens]
    nb = sum(need) + spare
    order = rng.permutation(nb)
    table = np.full((len(lens), max(max(need), wide or 1)), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    k = rng.integers(1, 256, (nb, n_kv, BLOCK, dim))
    v = rng.integers(1, 256, (nb, n_kv, BLOCK, dim))
    ks = rng.uniform(0.002, 0.03, (nb, n_kv)).astype(np.float32)
    vs = (10.0 ** rng.uniform(-3, 0, (nb, n_kv))).astype(np.float32)
    sums = (k - 128).sum(2).astype(np.int16)
    raw_k = k.reshape(nb, n_kv, BLOCK, dim // 64, 64).transpose(0, 1, 3, 2, 4)
    c = api.KvCache(T.from_numpy(np.ascontiguousarray(raw_k).astype(np.uint8)).cuda(),
                    T.from_numpy(np.ascontiguousarray(v.transpose(0, 1, 3, 2)).astype(np.uint8)).cuda(), T.from_numpy(ks).cuda(),
                    T.from_numpy(vs).cuda(), T.from_numpy(table).cuda(), T.from_numpy(sums).cuda())
    return c, dict(k=k, v=v, ks=ks, vs=vs, table=table, sums=sums)


def seq_values(host, s, n, h):
    """f64 keys and values [n, dim] of the first n tokens of sequence s."""
    ids = host["table"][s, :-(-n // BLOCK)]
    k = ((host["k"][ids, h] - 128) * host["ks"][ids, h].astype(np.float64)[:, None, None]).reshape(-1, host["k"].shape[-1])[:n]
    v = ((host["v"][ids, h] - 128) * host["vs"][ids, h].astype(np.float64)[:, None, None]).reshape(-1, host["k"].shape[-1])[:n]
    return k, v


def plain_attention(host, new, lens, q, n_kv, scale, window=0, sel=None, absent=()):
    """(out, lse, A, vmax) in f64; absent: (sequence, block) pairs the table does not have."""
    N, H, D = q.shape
    G = H // n_kv
    out, lse = np.zeros((N, H, D)), np.full((N, H), -np.inf)
    A, vmax = np.zeros((N, H)), np.zeros((N, H))
    row = 0
    for s, (m, n) in enumerate(zip(new, lens)):
        for i in range(m):
            pos = n - m + i
            for h in range(n_kv):
                j = np.arange(max(pos + 1, 0))
                if window:
                    j = j[j > pos - window]
                if sel is not None:
                    j = j[np.isin(j // BLOCK, sel[row + i, h])]
                for b in [b for t, b in absent if t == s]:
                    j = j[j // BLOCK != b]
                if len(j) == 0:
                    continue
                k, v = seq_values(host, s, n, h)
                k, v = k[j], v[j]
                for g in range(G):
                    x = q[row + i, h * G + g]
                    z = scale * (k @ x)
                    top = z.max()
                    p = np.exp(z - top)
                    out[row + i, h * G + g] = p @ v / p.sum()
                    lse[row + i, h * G + g] = top + np.log(p.sum())
                    A[row + i, h * G + g] = scale * (np.abs(k) @ np.abs(x)).max()
                    vmax[row + i, h * G + g] = np.abs(v).max()
        row += m
    return out, lse, A, vmax


def check(got, lse, want, bf16):
    out, ref_lse, A, vmax = want
    tol = (2 * 2.0 ** -20 * A + 2.0 ** -19) * vmax
    if bf16:
        tol = tol + 2.0 ** -11 * vmax
    tol = tol[..., None] + (2.0 ** -8 * np.abs(out) if bf16 else 0)
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    bad = np.abs(got - out) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], (np.abs(got - out) / np.maximum(tol, 1e-30)).max())
    if lse is not None:
        lse = lse.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isneginf(lse), np.isneginf(ref_lse))
        fin = np.isfinite(ref_lse)
        assert (np.abs(lse[fin] - ref_lse[fin]) <= 2 * 2.0 ** -20 * A[fin] + 2.0 ** -19 + 2.0 ** -22 * np.abs(ref_lse[fin])).all()


def attend(T, cache, new, lens, q, window=0, sel=None, scale=None, attn=None, lse=True):
    from project_maya_b200 import api
    batch = api.AttnBatch.of(new, lens)
    attn = attn or api.KvAttention(cache, q.shape[1], window=window, scale=scale)
    l = T.full(q.shape[:2], 7.0, dtype=T.float32, device="cuda") if lse else None
    out = attn.forward(batch, q, sel=sel, out=T.full(q.shape, 7.0, dtype=q.dtype, device="cuda"), lse=l)
    T.cuda.synchronize()
    assert attn.error() == 0
    return out, l


CASES = [
    # new tokens, lengths, key/value heads, group, head size, window
    ([1], [1], 1, 1, 64, 0),
    ([1], [64], 2, 4, 128, 0),
    ([1, 1, 1], [65, 63, 1000], 2, 5, 128, 0),
    ([1, 1], [700, 129], 2, 16, 256, 0),
    ([1], [515], 1, 20, 64, 0),              # a group beyond 16 heads: two rings of 32 rows
    ([1], [200], 1, 40, 192, 0),             # 64 rows
    ([1], [300], 1, 71, 128, 0),             # more rows than a tile has
    ([3, 0, 2], [10, 0, 200], 3, 3, 128, 0),  # a sequence of no tokens
    ([4], [2], 2, 2, 64, 0),                 # more new tokens than the sequence holds: two rows see nothing
    ([8, 8], [100, 1030], 2, 8, 64, 0),
    ([8], [333], 1, 7, 256, 0),
    ([70], [70], 2, 1, 128, 0),
    ([33, 90], [400, 90], 1, 6, 128, 0),
    ([20], [500], 1, 3, 192, 0),
    ([1, 1], [1000, 40], 2, 4, 128, 100),
    ([9, 30], [400, 30], 2, 2, 64, 65),
    ([5], [200], 1, 4, 256, 1),              # each token sees itself alone
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(cuda, case, bf16):
    import torch as T
    new, lens, n_kv, group, dim, window = CASES[case]
    rng = np.random.default_rng(100 + case)
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    q = T.from_numpy(rng.standard_normal((sum(new), n_kv * group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    want = plain_attention(host, new, lens, q.double().numpy(), n_kv, dim ** -0.5, window)
    out, lse = attend(T, cache, new, lens, q.cuda(), window)
    check(out, lse, want, bf16)


@pytest.mark.parametrize("bf16", [False, True])
def test_long_sequence_is_split_and_joined(cuda, bf16):
    import torch as T
    rng = np.random.default_rng(5)
    lens, new = [20011, 37], [1, 1]
    cache, host = make_cache(T, rng, lens, 1, 128)
    q = T.from_numpy(rng.standard_normal((2, 4, 128)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    want = plain_attention(host, new, lens, q.double().numpy(), 1, 128 ** -0.5)
    out, lse = attend(T, cache, new, lens, q.cuda())
    check(out, lse, want, bf16)
    again, _ = attend(T, cache, new, lens, q.cuda())
    assert T.equal(out, again)                # whichever split is last


PROMPTS = [
    # the same columns; 128 rows (tokens * group) of a sequence and more in bf16: the tensor-core kernel's tiles of 256
    ([128], [128], 1, 1, 128, 0),
    ([129], [129], 2, 1, 64, 0),
    ([256], [300], 1, 1, 128, 0),
    ([43, 0, 100, 1], [43, 70, 1000, 900], 2, 6, 128, 0),
    ([300], [300], 1, 2, 64, 0),
    ([130], [64], 1, 1, 128, 0),             # 66 rows before the sequence: one tile sees nothing at all
    ([200], [777], 1, 3, 128, 130),
    ([257, 20], [257, 300], 1, 7, 64, 64),
    ([17], [2100], 1, 16, 128, 0),
    ([150], [400], 1, 1, 128, 1),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts(cuda, case, bf16):
    import torch as T
    new, lens, n_kv, group, dim, window = PROMPTS[case]
    rng = np.random.default_rng(400 + case)
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    q = T.from_numpy(rng.standard_normal((sum(new), n_kv * group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    want = plain_attention(host, new, lens, q.double().numpy(), n_kv, dim ** -0.5, window)
    out, lse = attend(T, cache, new, lens, q.cuda(), window)
    check(out, lse, want, bf16)
    again, _ = attend(T, cache, new, lens, q.cuda(), window, lse=False)
    assert T.equal(out, again)


@pytest.mark.parametrize("dim,window", [(128, 0), (64, 0), (128, 2500)])
def test_few_prompt_rows_over_a_long_context(cuda, dim, window):
    """A tile or two a head over many blocks: cut into pieces that are joined; a sequence so short that some of its pieces are empty, one of no tokens."""
    import torch as T
    rng = np.random.default_rng(50 + dim)
    new, lens, n_kv, group = [50, 50, 0, 60], [7000, 90, 300, 40], 2, 3                # (the last: 20 rows before the sequence)
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    q = T.from_numpy(rng.standard_normal((160, n_kv * group, dim)).astype(np.float32)).bfloat16()
    out, lse = attend(T, cache, new, lens, q.cuda(), window)
    check(out, lse, plain_attention(host, new, lens, q.double().numpy(), n_kv, dim ** -0.5, window), True)
    again, _ = attend(T, cache, new, lens, q.cuda(), window, lse=False)
    assert T.equal(out, again)


def test_prompt_with_large_scores_and_scales_far_apart(cuda):
    """Rows whose maximum rises late and by much, value scales 1e-20 .. 1 and 0, blocks the table does not have, unaligned queries."""
    import torch as T
    rng = np.random.default_rng(17)
    lens, new = [1000], [160]
    cache, host = make_cache(T, rng, lens, 1, 128)
    for b in range(16):
        host["ks"][host["table"][0, b]] = 0.002 * 1.3 ** b
        host["vs"][host["table"][0, b]] = (0.0, 1e-20, 1.0, 1e-3)[b % 4]
    cache.k_scale.copy_(T.from_numpy(host["ks"]))
    cache.v_scale.copy_(T.from_numpy(host["vs"]))
    rows = T.from_numpy(4 * rng.standard_normal((160, 131)).astype(np.float32)).bfloat16().cuda()
    for off in (0, 3):
        q = rows[:, off:off + 128].unflatten(1, (1, 128))
        out, lse = attend(T, cache, new, lens, q)
        check(out, lse, plain_attention(host, new, lens, q.double().cpu().numpy(), 1, 128 ** -0.5), True)
    cache.table[0, 3] = -1
    cache.table[0, 8:10] = cache.n_blocks
    out, lse = attend(T, cache, new, lens, q)
    check(out, lse, plain_attention(host, new, lens, q.double().cpu().numpy(), 1, 128 ** -0.5, absent=((0, 3), (0, 8), (0, 9))), True)


@pytest.mark.parametrize("bf16,dim,group", [(True, 128, 4), (False, 64, 9), (True, 256, 2), (False, 128, 8)])
def test_many_sequences(cuda, bf16, dim, group):
    """More sequences than a thread block adds up: one a thread block, in one piece, the long one over several look-ups of its blocks."""
    import torch as T
    rng = np.random.default_rng(30 + group)
    lens = [int(n) for n in rng.integers(0, 200, 300)]
    lens[5], lens[17], lens[299] = 0, 9000, 64
    new = [1] * 300
    cache, host = make_cache(T, rng, lens, 1, dim)
    q = T.from_numpy(rng.standard_normal((300, group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    out, lse = attend(T, cache, new, lens, q.cuda())
    check(out, lse, plain_attention(host, new, lens, q.double().numpy(), 1, dim ** -0.5), bf16)


def test_many_heads_and_sequences(cuda):
    """So many (sequence, head)s that there is no room for parts of them: none is cut."""
    import torch as T
    rng = np.random.default_rng(40)
    lens, n_kv = [int(n) for n in rng.integers(1, 300, 240)], 16
    cache, host = make_cache(T, rng, lens, n_kv, 64)
    q = T.from_numpy(rng.standard_normal((240, n_kv, 64)).astype(np.float32)).bfloat16()
    out, lse = attend(T, cache, [1] * 240, lens, q.cuda())
    check(out, lse, plain_attention(host, [1] * 240, lens, q.double().numpy(), n_kv, 0.125), True)


def test_long_f32_prompt(cuda):
    """Rows that fill more than 256 tiles: first, middle and last tokens."""
    import torch as T
    rng = np.random.default_rng(41)
    n, group, dim = 2200, 8, 64
    cache, host = make_cache(T, rng, [n], 1, dim)
    q = T.from_numpy(rng.standard_normal((n, group, dim)).astype(np.float32)).cuda()
    out, lse = attend(T, cache, [n], [n], q)
    for a in (0, 1000, n - 8):
        want = plain_attention(host, [8], [a + 8], q[a:a + 8].double().cpu().numpy(), 1, dim ** -0.5)
        check(out[a:a + 8], lse[a:a + 8], want, False)


def test_long_lists_of_many_tokens(cuda):
    """Lists longer than one look-up of their blocks, a warp each."""
    import torch as T
    rng = np.random.default_rng(42)
    n, new, n_kv, n_sel = 13000, 1800, 4, 150
    cache, host = make_cache(T, rng, [n], n_kv, 64)
    sel = np.sort(np.argsort(rng.random((new, n_kv, (n - new) // BLOCK)), -1)[..., :n_sel], -1).astype(np.int32)
    q = T.from_numpy(rng.standard_normal((new, n_kv * 2, 64)).astype(np.float32)).cuda()
    out, lse = attend(T, cache, [new], [n], q, sel=T.from_numpy(sel).cuda())
    for a in (0, new - 5):
        end = n - new + a + 5
        want = plain_attention(host, [5], [end], q[a:a + 5].double().cpu().numpy(), n_kv, 0.125, sel=sel[a:a + 5])
        check(out[a:a + 5], lse[a:a + 5], want, False)


def test_strided_and_unaligned_queries(cuda):
    import torch as T
    rng = np.random.default_rng(6)
    lens, new = [90, 200], [2, 3]
    cache, host = make_cache(T, rng, lens, 2, 128)
    rows = T.from_numpy(rng.standard_normal((5, 3 + 10 * 128)).astype(np.float32)).cuda()
    for off in (0, 1, 3):
        q = rows[:, off:off + 8 * 128].unflatten(1, (8, 128))
        want = plain_attention(host, new, lens, q.double().cpu().numpy(), 2, 128 ** -0.5)
        out, lse = attend(T, cache, new, lens, q)
        check(out, lse, want, False)


def test_scores_of_any_size(cuda):
    """Scores in the hundreds (one token takes all), queries of 1e-30 and 1e30, zero queries, blocks whose scale is 0."""
    import torch as T
    rng = np.random.default_rng(7)
    lens, new = [300], [4]
    cache, host = make_cache(T, rng, lens, 1, 64)
    host["ks"][host["table"][0, 1]] = 0
    host["vs"][host["table"][0, 2]] = 0
    cache.k_scale.copy_(T.from_numpy(host["ks"]))
    cache.v_scale.copy_(T.from_numpy(host["vs"]))
    x = rng.standard_normal((4, 2, 64))
    x[0] *= 300
    x[1, 0] *= 1e-30
    x[2, 0] = 0
    q = T.from_numpy(x.astype(np.float32))
    out, lse = attend(T, cache, new, lens, q.cuda())
    check(out, lse, plain_attention(host, new, lens, q.double().numpy(), 1, 0.125), False)
    q[3] *= 1e30
    out, _ = attend(T, cache, new, lens, q.cuda(), scale=0.125e-30)
    want = plain_attention(host, new, lens, q.double().numpy(), 1, 0.125e-30)
    check(out, None, want, False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group,dim", [(4, 128), (8, 64), (20, 128), (1, 256)])
def test_selected_blocks(cuda, group, dim, bf16):
    import torch as T
    rng = np.random.default_rng(8 + group)
    lens, new, n_kv, n_sel = [1500, 90, 700], [1, 2, 80], 2, 5
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    N = sum(new)
    sel = np.full((N, n_kv, n_sel), -1, np.int32)
    row = 0
    for m, n in zip(new, lens):
        for i in range(m):
            own = (n - m + i) // BLOCK
            for h in range(n_kv):
                k = rng.integers(0, min(n_sel, own + 1) + 1)                  # none at all among them
                sel[row, h, :k] = np.sort(rng.permutation(own + 1)[:k])
            row += 1
    sel[0, 0] = [-7, 3, 23, 24, 10 ** 9]                                      # beyond the sequence, beyond the table: passed over
    q = T.from_numpy(rng.standard_normal((N, n_kv * group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    want = plain_attention(host, new, lens, q.double().numpy(), n_kv, dim ** -0.5, sel=sel)
    out, lse = attend(T, cache, new, lens, q.cuda(), sel=T.from_numpy(sel).cuda())
    check(out, lse, want, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group,dim", [(8, 128), (3, 64), (1, 256), (5, 192)])
def test_selected_blocks_of_many_tokens(cuda, group, dim, bf16):
    """A prompt's lists, a warp each: the first tokens, some in the middle, the last."""
    import torch as T
    rng = np.random.default_rng(20 + group)
    n, n_kv, n_sel = 1900, 4, 6
    cache, host = make_cache(T, rng, [n], n_kv, dim)
    own = np.arange(n) // BLOCK
    sel = np.sort(np.where(rng.random((n, n_kv, n_sel)) < 0.8, np.floor(rng.random((n, n_kv, n_sel)) * (own[:, None, None] + 1)), -1).astype(np.int32), -1)
    sel[:, :, 1:][sel[:, :, 1:] == sel[:, :, :-1]] = -1                      # each block once
    sel[7] = -1                                                              # a row that sees nothing
    q = T.from_numpy(rng.standard_normal((n, n_kv * group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32).cuda()
    s = T.from_numpy(sel).cuda()
    out, lse = attend(T, cache, [n], [n], q, sel=s)
    assert (out[7] == 0).all()
    for a in (0, 640, 1860):
        want = plain_attention(host, [40], [a + 40], q[a:a + 40].double().cpu().numpy(), n_kv, dim ** -0.5, sel=sel[a:a + 40])
        check(out[a:a + 40], lse[a:a + 40], want, bf16)


def test_blocks_the_table_does_not_have(cuda):
    import torch as T
    rng = np.random.default_rng(9)
    lens, new = [400], [3]
    cache, host = make_cache(T, rng, lens, 1, 64)
    cache.table[0, 2] = -1
    cache.table[0, 4] = cache.n_blocks
    q = T.from_numpy(rng.standard_normal((3, 2, 64)).astype(np.float32))
    out, lse = attend(T, cache, new, lens, q.cuda())
    check(out, lse, plain_attention(host, new, lens, q.double().numpy(), 1, 0.125, absent=((0, 2), (0, 4))), False)


def test_lengths_beyond_the_bounds_are_held_to_them(cuda):
    """kv_len above max_len on the device: the rest is not read (nor anything outside)."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(10)
    cache, host = make_cache(T, rng, [256], 1, 64)
    q = T.from_numpy(rng.standard_normal((1, 1, 64)).astype(np.float32))
    batch = api.AttnBatch(T.tensor([0, 1], dtype=T.int32, device="cuda"), T.tensor([10 ** 6], dtype=T.int32, device="cuda"), 1, 1, 256)
    out = api.KvAttention(cache, 1).forward(batch, q.cuda())
    check(out, None, plain_attention(host, [1], [256], q.double().numpy(), 1, 0.125), False)


def test_cache_beyond_32_bit_offsets(cuda):
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(11)
    n_kv, dim, lens = 8, 256, [130, 70]
    small, host = make_cache(T, rng, lens, n_kv, dim)
    far = 33000                                                               # 33000 * 8 * 16 KB = 4.3e9 bytes
    n = small.n_blocks
    table = T.where(small.table >= 0, small.table + far, -1).int()
    big = api.KvCache.empty(far + n, n_kv, dim, table)
    for a, b in ((big.k, small.k), (big.v, small.v), (big.k_scale, small.k_scale), (big.v_scale, small.v_scale), (big.k_sum, small.k_sum)):
        a[far:].copy_(b)
    q = T.from_numpy(rng.standard_normal((2, n_kv, dim)).astype(np.float32))
    want = plain_attention(host, [1, 1], lens, q.double().numpy(), n_kv, dim ** -0.5)
    out, lse = attend(T, big, [1, 1], lens, q.cuda())
    check(out, lse, want, False)
    x = T.randn((2, n_kv, dim), device="cuda")
    for c in (big, small):                                                    # the append lands in the same codes
        api.KvAttention(c, n_kv).append(api.AttnBatch.of([1, 1], lens), q.cuda(), x, x, api.Rope())
    assert T.equal(big.k[far:], small.k) and T.equal(big.v[far:], small.v) and T.equal(big.k_sum[far:], small.k_sum)


def test_another_stream_and_a_graph(cuda):
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(12)
    lens, new = [3000, 64], [1, 1]
    cache, host = make_cache(T, rng, lens, 2, 128)
    q = T.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda()
    attn, batch = api.KvAttention(cache, 8), api.AttnBatch.of(new, lens)
    want = attn.forward(batch, q)
    out = T.zeros_like(want)
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    attn.forward(batch, q, out=out, stream=side)
    T.cuda.current_stream().wait_stream(side)
    assert T.equal(out, want)
    graph, out2 = T.cuda.CUDAGraph(), T.zeros_like(want)
    with T.cuda.graph(graph):
        attn.forward(batch, q, out=out2)
    for _ in range(3):
        out2.zero_()
        graph.replay()
        T.cuda.synchronize()
        assert T.equal(out2, want)


# ---------------------------------------------------------------- append
def plain_rows(x, w, cos, sin, pos, eps, pairs):
    x = x.astype(np.float64).copy()
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is not None:
        half = cos.shape[1]
        c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
        a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if pairs else (x[..., :half], x[..., half:2 * half])
        y, z = a * c - b * s, b * c + a * s
        if pairs:
            x[..., 0:2 * half:2], x[..., 1:2 * half:2] = y, z
        else:
            x[..., :half], x[..., half:2 * half] = y, z
    return x


def unpack(cache):
    k = cache.k.cpu().numpy().transpose(0, 1, 3, 2, 4)
    k = k.reshape(*k.shape[:3], -1).astype(np.int64) - 128
    return k, cache.v.cpu().numpy().transpose(0, 1, 3, 2).astype(np.int64) - 128


APPENDS = [
    # new tokens, lengths, key/value heads, group, head size, rotated, pairs, norms
    ([1], [1], 1, 1, 64, 64, False, True),
    ([1, 1, 1], [64, 65, 130], 2, 4, 128, 128, False, True),
    ([1, 0, 16], [7, 90, 70], 3, 5, 128, 64, True, True),
    ([130, 65], [130, 200], 2, 2, 64, 64, True, False),
    ([64, 3], [128, 3], 1, 8, 256, 128, False, True),
    ([63], [100], 1, 3, 192, 6, False, True),
    ([20], [20], 2, 1, 128, 0, False, True),
    ([5], [3], 1, 2, 64, 64, False, True),       # the first two tokens stand before the sequence: turned, not kept
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(cuda, case, bf16):
    import torch as T
    from project_maya_b200 import api
    new, lens, n_kv, group, dim, rot, pairs, norm = APPENDS[case]
    rng = np.random.default_rng(200 + case)
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    host_sum = cache.k_sum
    for s, (m, n) in enumerate(zip(new, lens)):              # k_sum of what was there before
        for b in range(-(-n // BLOCK)):
            held = max(0, min(BLOCK, n - m - b * BLOCK))
            host_sum[int(host["table"][s, b])] = T.from_numpy((host["k"][host["table"][s, b], :, :held] - 128).sum(1).astype(np.int16)).cuda()
    before_k, before_v = unpack(cache)
    ks0, vs0 = host["ks"].copy(), host["vs"].copy()
    N, H = sum(new), n_kv * group
    dt = T.bfloat16 if bf16 else T.float32
    wide = T.from_numpy(rng.standard_normal((N, (H + 2 * n_kv) * dim + 8)).astype(np.float32)).to(dt).cuda()
    q, k, v = wide[:, :(H + 2 * n_kv) * dim].unflatten(1, (-1, dim)).split((H, n_kv, n_kv), 1)
    angle = np.arange(max(lens))[:, None] * 100.0 ** (-np.arange(max(rot // 2, 1)) / max(rot // 2, 1))
    cos, sin = (np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)) if rot else (None, None)
    qw, kw = (1 + 0.1 * rng.standard_normal((2, dim)).astype(np.float32)) if norm else (None, None)
    dev = lambda x: None if x is None else T.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
    rope = api.Rope(dev(cos), dev(sin), dev(qw), dev(kw), eps=1e-5, pairs=pairs)
    q_out = api.KvAttention(cache, H).append(api.AttnBatch.of(new, lens), q, k, v, rope)
    T.cuda.synchronize()
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lens)]).astype(int)
    turn = np.clip(pos, 0, None)
    q_want = plain_rows(q.double().cpu().numpy(), qw, cos, sin, turn, 1e-5, pairs)
    got = q_out.double().cpu().numpy()
    # f32: a norm (sum of `dim` squares, a reciprocal root) and two products: within 2^-20 of the row's largest
    tol = 2.0 ** -20 * np.abs(q_want).max(-1, keepdims=True) + (2.0 ** -8 * np.abs(q_want) if bf16 else 0)
    assert (np.abs(got - q_want) <= tol).all()
    after_k, after_v = unpack(cache)
    ks1, vs1, sums = cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy(), cache.k_sum.cpu().numpy()
    touched = set()
    for name, x, before, after, s0, s1 in (("k", plain_rows(k.double().cpu().numpy(), kw, cos, sin, turn, 1e-5, pairs), before_k, after_k, ks0, ks1),
                                          ("v", v.double().cpu().numpy(), before_v, after_v, vs0, vs1)):
        row = 0
        for s, (m, n) in enumerate(zip(new, lens)):
            for b in range(max(n - m, 0) // BLOCK if m else 0, -(-n // BLOCK) if m else 0):
                held, end = max(0, n - m - b * BLOCK), min(BLOCK, n - b * BLOCK)
                at = row + b * BLOCK + held - (n - m)
                phys = host["table"][s, b]
                touched.add(phys)
                for h in range(n_kv):
                    fresh = x[at:at + end - held, h]
                    old = float(s0[phys, h]) if held else 0.0
                    want = max(old, np.abs(fresh).max() / 127)
                    scale = float(s1[phys, h])
                    assert abs(scale - want) <= 2.0 ** -20 * want
                    codes = after[phys, h]
                    # nearest: half a step, and what the row itself may be off
                    assert (np.abs(codes[held:end] * scale - fresh) <= scale * (0.5 + 127 * 2.0 ** -19)).all()
                    moved = before[phys, h, :held] * (old / scale) if scale > old else before[phys, h, :held]
                    assert (np.abs(codes[:held] - moved) <= 0.5 + 2.0 ** -14).all() and (scale > old or np.array_equal(codes[:held], moved))
                    assert np.array_equal(codes[end:], before[phys, h, end:])            # nothing behind the last token
                    if name == "k":
                        assert np.array_equal(sums[phys, h], codes[:end].sum(0))
            row += m
    rest = [b for b in range(cache.n_blocks) if b not in touched]
    assert np.array_equal(after_k[rest], before_k[rest]) and np.array_equal(after_v[rest], before_v[rest])
    assert np.array_equal(ks1[rest], ks0[rest]) and np.array_equal(vs1[rest], vs0[rest])


def test_append_one_by_one_stays_near_one_pass(cuda):
    """64 tokens appended singly: a code is rounded once more at each growth of its block's scale - within (growths + 1) / 2 steps."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(3)
    n_kv, dim = 2, 64
    x = T.randn((64, n_kv, dim), device="cuda")
    table = T.zeros((1, 1), dtype=T.int32, device="cuda")
    cache = api.KvCache.empty(1, n_kv, dim, table)
    attn, grown = api.KvAttention(cache, n_kv), T.zeros((1, n_kv), device="cuda")
    last = None
    for i in range(64):
        attn.append(api.AttnBatch.of([1], [i + 1]), x[i:i + 1], x[i:i + 1], x[i:i + 1], api.Rope())
        if last is not None:
            grown += cache.v_scale > last
        last = cache.v_scale.clone()
    _, v, mean = cache.read(table[0], dtype=T.float32)
    step = cache.v_scale[0][None, :, None]
    assert ((v[0] - x).abs() <= step * ((grown[0][None, :, None] + 1) / 2 + 1e-3)).all()
    k = cache.k[0].transpose(1, 2).flatten(2).int() - 128                     # [n_kv, token, dim]
    assert T.equal(cache.k_sum[0].int(), k.sum(1).int())
    assert T.allclose(mean[0], k.float().sum(1) * cache.k_scale[0][:, None] / 64, rtol=1e-6, atol=0)


def test_append_after_tokens_were_taken_back(cuda):
    """A window of draft tokens, cut short, and another in its place: the sums are of what the block holds now."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(4)
    cache = api.KvCache.empty(2, 2, 64, T.tensor([[1, 0]], dtype=T.int32, device="cuda"))
    attn = api.KvAttention(cache, 2)
    for new, length, size in ((40, 40, 1.0), (8, 48, 1.0), (8, 44, 0.5), (8, 52, 3.0), (16, 64, 0.1), (4, 64, 1.0)):
        x = size * T.randn((new, 2, 64), device="cuda")
        attn.append(api.AttnBatch.of([new], [length]), x, x, x, api.Rope())
        k = cache.k[1].transpose(1, 2).flatten(2).int()[:, :length] - 128
        assert T.equal(cache.k_sum[1].int(), k.sum(1).int())


def test_append_not_finite(cuda):
    import torch as T
    from project_maya_b200 import api
    cache = api.KvCache.empty(2, 1, 64, T.tensor([[0], [1]], dtype=T.int32, device="cuda"))
    x = T.ones((2, 1, 64), device="cuda")
    x[0, 0, 3], x[0, 0, 4], x[1, 0, 5] = float("inf"), float("-inf"), float("nan")
    api.KvAttention(cache, 1).append(api.AttnBatch.of([1, 1], [1, 1]), T.ones_like(x), x, x, api.Rope())
    _, v = unpack(cache)
    assert v[0, 0, 0, 3] == 127 and v[0, 0, 0, 4] == -127 and abs(float(cache.v_scale[0, 0]) / 1e30 - 1) < 1e-6
    assert v[1, 0, 0, 5] == 0 and v[1, 0, 0, 0] == 127


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_read(cuda, dim, dtype):
    import torch as T
    rng = np.random.default_rng(13)
    cache, host = make_cache(T, rng, [300], 3, dim)
    ids, counts = np.array([2, 0, 4, -1, cache.n_blocks], np.int32), np.array([64, 1, 33, 64, 5], np.int32)
    for c in (counts, None):
        k, v, mean = cache.read(T.from_numpy(ids).cuda(), None if c is None else T.from_numpy(c).cuda(), dtype=getattr(T, dtype))
        for i, b in enumerate(ids):
            n = 0 if not 0 <= b < cache.n_blocks else 64 if c is None else c[i]
            for got, which in ((k, "k"), (v, "v")):
                want = np.zeros((64, 3, dim), np.float32)
                if n:
                    want[:n] = ((host[which][b, :, :n] - 128).astype(np.float32) * host[which + "s"][b][:, None, None]).transpose(1, 0, 2)
                assert T.equal(got[i].cpu(), T.from_numpy(want).to(getattr(T, dtype)))
            want = host["sums"][b].astype(np.float32) * host["ks"][b][:, None] / np.float32(n) if n else np.zeros((3, dim), np.float32)
            assert T.equal(mean[i].cpu(), T.from_numpy(want).to(getattr(T, dtype)))


# ---------------------------------------------------------------- selection
def plain_select(host, new, lens, q, n_kv, n_sel, n_first, n_last):
    """The rule in whole numbers and one f32 product after the other: the same lists, bit for bit."""
    N, H, D = q.shape
    G = H // n_kv
    scale = np.abs(q).max(-1, keepdims=True) * np.float32(1 / 127)
    q8 = np.where(scale > 0, np.clip(np.rint(q / np.where(scale > 0, scale, 1)), -127, 127), 0).astype(np.int64)
    out = np.full((N, n_kv, n_sel), -1, np.int32)
    row = 0
    for s, (m, n) in enumerate(zip(new, lens)):
        for i in range(m):
            own = (n - m + i) // BLOCK
            if n - m + i < 0:
                continue
            ids = host["table"][s, :own + 1]
            for h in range(n_kv):
                dots = q8[row + i, h * G:(h + 1) * G] @ host["sums"][ids, h].astype(np.int64).T
                sc = (dots.astype(np.float32) * scale[row + i, h * G:(h + 1) * G] * host["ks"][ids, h]).max(0)
                b = np.arange(own + 1)
                sc = np.where((b < n_first) | (b > own - n_last), np.inf, sc)
                pick = np.sort(np.argsort(-sc, kind="stable")[:n_sel])
                out[row + i, h, :len(pick)] = pick
        row += m
    return out


SELECTS = [
    # new tokens, lengths, key/value heads, group, head size, selected, first, last
    ([1], [1], 1, 1, 64, 1, 0, 1),
    ([1], [64], 2, 4, 128, 4, 1, 2),
    ([1, 1, 0], [1300, 320, 65], 2, 8, 128, 6, 1, 2),
    ([1], [70000], 1, 8, 128, 32, 1, 1),         # shared out over a cluster
    ([1], [9000], 2, 5, 256, 17, 0, 1),
    ([5], [3], 1, 2, 64, 3, 0, 1),               # tokens before the sequence
    ([90, 33], [2000, 33], 2, 3, 64, 9, 2, 3),
    ([40], [3000], 1, 16, 192, 20, 1, 1),
    ([3], [2500], 1, 40, 128, 12, 1, 1),         # a group beyond 16 heads
    ([200], [5000], 1, 1, 128, 30, 1, 2),
    ([1], [40000], 1, 12, 64, 512, 3, 4),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("case", range(len(SELECTS)))
def test_select(cuda, case, bf16):
    import torch as T
    from project_maya_b200 import api
    new, lens, n_kv, group, dim, n_sel, n_first, n_last = SELECTS[case]
    rng = np.random.default_rng(300 + case)
    cache, host = make_cache(T, rng, lens, n_kv, dim)
    q = T.from_numpy(rng.standard_normal((sum(new), n_kv * group, dim)).astype(np.float32)).to(T.bfloat16 if bf16 else T.float32)
    attn = api.KvAttention(cache, n_kv * group, n_sel=n_sel, n_first=n_first, n_last=n_last)
    sel = attn.select(api.AttnBatch.of(new, lens), q.cuda(), sel=T.full((sum(new), n_kv, n_sel), -5, dtype=T.int32, device="cuda"))
    assert np.array_equal(sel.cpu().numpy(), plain_select(host, new, lens, q.float().numpy(), n_kv, n_sel, n_first, n_last))


def test_select_equal_scores_take_the_lowest_blocks(cuda):
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(14)
    for lens in ([4000], [60000]):
        cache, host = make_cache(T, rng, lens, 1, 64)
        host["sums"][:] = rng.integers(-1, 2, (cache.n_blocks, 1, 1))         # three scores in all
        host["ks"][:] = 0.5
        cache.k_sum.copy_(T.from_numpy(host["sums"]))
        cache.k_scale.fill_(0.5)
        for x in (T.ones((1, 2, 64)), T.zeros((1, 2, 64))):
            sel = api.KvAttention(cache, 2, n_sel=11, n_first=1, n_last=1).select(api.AttnBatch.of([1], lens), x.cuda())
            assert np.array_equal(sel.cpu().numpy(), plain_select(host, [1], lens, x.numpy(), 1, 11, 1, 1))


def test_select_then_attend_over_every_block_is_attention(cuda):
    """With as many entries as blocks the list is all of them: the same result as without one."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(15)
    lens, new = [500, 100], [1, 1]
    cache, _ = make_cache(T, rng, lens, 2, 128)
    q = T.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda()
    attn, batch = api.KvAttention(cache, 8, n_sel=8), api.AttnBatch.of(new, lens)
    sel = attn.select(batch, q)
    a, b = attn.forward(batch, q, sel=sel), attn.forward(batch, q)
    assert T.allclose(a, b, rtol=0, atol=2.0 ** -18 * float(b.abs().max()) * 8)


# ---------------------------------------------------------------- refusals
def test_refusals_launch_nothing(cuda):
    import torch as T
    from project_maya_b200 import _lib, api
    rng = np.random.default_rng(16)
    cache, _ = make_cache(T, rng, [100], 2, 64)
    q = T.zeros((1, 4, 64), device="cuda")
    batch = api.AttnBatch.of([1], [100])
    launches = _lib.load().maya_launch_count()
    for kw, status in ((dict(window=-1), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1)):
        with pytest.raises(api.MayaError) as e:
            api.KvAttention(cache, 4, **kw).forward(batch, q)
        assert e.value.status == status
    with pytest.raises(api.MayaError):                                        # heads that are no whole groups
        api.KvAttention(cache, 3)
    with pytest.raises(api.MayaError) as e:                                   # longer than the table
        api.KvAttention(cache, 4).forward(api.AttnBatch.of([1], [129]), q)
    assert e.value.status == -1
    with pytest.raises(api.MayaError) as e:
        api.KvAttention(cache, 4).forward(batch, q, sel=T.zeros((1, 2, 513), dtype=T.int32, device="cuda"))
    assert e.value.status == -4
    for kw, status in ((dict(n_sel=2, n_first=1, n_last=2), -1), (dict(n_sel=2, n_first=0, n_last=0), -1), (dict(n_sel=513), -4), (dict(n_sel=0), -1)):
        with pytest.raises(api.MayaError) as e:
            api.KvAttention(cache, 4, **kw).select(batch, q)
        assert e.value.status == status
    bare = api.KvCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.table)
    with pytest.raises(api.MayaError):                                        # no sums to select by
        api.KvAttention(bare, 4, n_sel=4).select(batch, q)
    with pytest.raises(api.MayaError):                                        # angles for 66 of 64 values
        api.KvAttention(cache, 4).append(batch, q, q[:, :2], q[:, :2], api.Rope(T.zeros((100, 33), device="cuda"), T.zeros((100, 33), device="cuda")))
    with pytest.raises(AssertionError):
        api.KvAttention(cache, 4).forward(batch, q.half())
    assert _lib.load().maya_launch_count() == launches
    nothing = api.AttnBatch.of([0], [100])                                    # no new tokens: nothing to do
    assert api.KvAttention(cache, 4).forward(nothing, q[:0]).shape == (0, 4, 64)
    assert _lib.load().maya_launch_count() == launches
