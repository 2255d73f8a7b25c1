"""Blocks of the cache reserved, forked, freed, compacted and copied on the device, against the same done one by one on the host.  Whole numbers and moved
bytes: everything is equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
BLOCK = 64
PARTS = ("k", "v", "k_scale", "v_scale", "k_sum")


class Host:
    """The caches, the table and the counts on the host, and every call one by one."""

    def __init__(self, rng, n_seq, wide, n_blocks, layers=1, kv=1, dim=64, sums=True):
        self.nb, self.sums = n_blocks, sums
        self.layers = [dict(k=rng.integers(0, 256, (n_blocks, kv, dim // 64, BLOCK, 64), dtype=np.uint8),
                            v=rng.integers(0, 256, (n_blocks, kv, dim, BLOCK), dtype=np.uint8),
                            k_scale=rng.random((n_blocks, kv), dtype=np.float32), v_scale=rng.random((n_blocks, kv), dtype=np.float32),
                            k_sum=rng.integers(-99, 99, (n_blocks, kv, dim)).astype(np.int16)) for _ in range(layers)]
        self.table = np.full((n_seq, wide), -1, np.int32)
        self.refs = np.zeros(n_blocks, np.int32)
        self.error = 0

    def fill(self, rng, lens):
        order = rng.permutation(self.nb)
        at = 0
        for s, n in enumerate(lens):
            for b in range(-(-n // BLOCK)):
                self.table[s, b] = order[at]
                self.refs[order[at]] = 1
                at += 1
        return self

    def device(self, T):
        from project_maya_b200 import api
        table = T.from_numpy(self.table).cuda()
        caches = []
        for p in self.layers:
            t = {n: T.from_numpy(p[n]).cuda() for n in PARTS}
            caches.append(api.KvCache(t["k"], t["v"], t["k_scale"], t["v_scale"], table, k_sum=t["k_sum"] if self.sums else None))
        return api.KvPages(caches, T.from_numpy(self.refs).cuda())

    def is_block(self, e):
        return 0 <= e < self.nb

    def take(self, free, n):
        if len(free) < n:
            self.error = 1
        return list(free[:n]) + [-1] * (n - len(free[:n]))

    def move(self, pairs):
        old = [{n: p[n].copy() for n in PARTS} for p in self.layers]
        for s, d in pairs:
            for p, o in zip(self.layers, old):
                for n in PARTS:
                    if n != "k_sum" or self.sums:
                        p[n][d] = o[n][s]

    def reserve(self, new, lens):
        items, free = [], np.flatnonzero(self.refs <= 0)
        for s, (m, n) in enumerate(zip(new, lens)):
            if m > 0 and n > 0:
                old = max(0, n - m)
                items += [(s, b, b * BLOCK < old) for b in range(old // BLOCK, (n - 1) // BLOCK + 1)]
        items = [(s, b, held) for s, b, held in items if not self.is_block(self.table[s, b]) or self.refs[self.table[s, b]] > 1]
        pairs = []
        for (s, b, held), f in zip(items, self.take(free, len(items))):
            e = self.table[s, b]
            if self.is_block(e):
                self.refs[e] -= 1
                if held and f >= 0:
                    pairs.append((e, f))
            if f >= 0:
                self.refs[f] = 1
            self.table[s, b] = f
        self.move(pairs)

    def fork(self, parents, children, lens):
        seen, jobs, S = set(), [], len(self.table)
        for p, c, n in zip(parents, children, lens):
            if 0 <= c < S and c not in seen:
                seen.add(c)
                if 0 <= p < S and p != c:
                    jobs.append((p, c, min(max(n, 0), self.table.shape[1] * BLOCK)))
        was, free = self.table.copy(), np.flatnonzero(self.refs <= 0)
        wants = [j for j in jobs if j[2] % BLOCK and self.is_block(was[j[0], j[2] // BLOCK])]
        got = dict(zip([j[1] for j in wants], self.take(free, len(wants))))
        pairs = []
        for p, c, n in jobs:
            full = n // BLOCK
            for e in was[c]:
                if self.is_block(e):
                    self.refs[e] -= 1
            row = np.full(self.table.shape[1], -1, np.int32)
            for b in range(full):
                if self.is_block(was[p, b]):
                    row[b] = was[p, b]
                    self.refs[row[b]] += 1
            if c in got:
                row[full] = got[c]
                if got[c] >= 0:
                    self.refs[got[c]] = 1
                    pairs.append((was[p, full], got[c]))
            self.table[c] = row
        self.move(pairs)

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.table):
                for e in self.table[s]:
                    if self.is_block(e):
                        self.refs[e] -= 1
                self.table[s] = -1

    def compact(self, most=None):
        live = int((self.refs > 0).sum())
        dst, src = np.flatnonzero(self.refs[:live] <= 0)[:most], live + np.flatnonzero(self.refs[live:] > 0)[:most]
        to = dict(zip(src.tolist(), dst.tolist()))
        self.table = np.array([[to.get(e, e) for e in row] for row in self.table.tolist()], np.int32)
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        self.move(list(zip(src, dst)))
        return live

    def same(self, T, pages):
        assert np.array_equal(pages.table.cpu().numpy(), self.table)
        assert np.array_equal(pages.refs.cpu().numpy(), self.refs)
        for c, p in zip(pages.caches, self.layers):
            for n in PARTS:
                if n != "k_sum" or self.sums:
                    assert np.array_equal(getattr(c, n).cpu().numpy(), p[n]), n
        assert pages.error() == self.error
        self.error = 0


def i32(T, v):
    return T.tensor(v, dtype=T.int32, device="cuda")


def batch_of(new, lens):
    from project_maya_b200 import api
    return api.AttnBatch.of(new, lens)


@pytest.mark.parametrize("layers,kv,dim,sums", [(1, 1, 64, True), (3, 2, 128, True), (2, 5, 192, False), (1, 8, 256, True)])
def test_a_serving_run(cuda, layers, kv, dim, sums):
    """Prompts, steps, forks, rollbacks, leavers and compactions in a row, everything compared after each call."""
    import torch as T
    rng = np.random.default_rng(dim + layers)
    host = Host(rng, 9, 7, 60, layers, kv, dim, sums)
    pages = host.device(T)
    lens = [0] * 9

    def reserve(new):
        for s, n in enumerate(new):
            lens[s] = min(lens[s] + n, 7 * BLOCK) if n else lens[s]
        host.reserve(new, lens)
        pages.reserve(batch_of(new, lens))
        host.same(T, pages)

    def fork(p, c, n):
        was = list(lens)
        host.fork(p, c, n)
        pages.fork(i32(T, p), i32(T, c), i32(T, n))
        for a, b, m in zip(p, c, n):
            if a != b:
                lens[b] = min(m, was[a])
        host.same(T, pages)

    reserve([130, 1, 64, 65, 0, 0, 0, 0, 0])
    reserve([1] * 4 + [0] * 5)
    fork([0, 0, 2, 3], [4, 5, 6, 3], [131, 128, 65, 66])
    reserve([1, 1, 1, 1, 1, 1, 1, 0, 0])
    fork([4, 0, 5, 6, 1, 2], [0, 4, 1, 2, 5, 6], [132, 132, 129, 66, 3, 66])       # a permutation among beams
    reserve([1] * 7 + [0, 0])
    fork([0, 0], [7, 8], [128, 64])
    lens[7] = 100                                                                  # taken back into a block that others hold
    reserve([0, 0, 0, 0, 0, 0, 0, 30, 1])
    host.free([2, 0, 5, 2])
    pages.free(i32(T, [2, 0, 5, 2]))
    lens[0] = lens[2] = lens[5] = 0
    host.same(T, pages)
    live = host.compact()
    pages.compact()
    host.same(T, pages)
    assert pages.live.item() == live == (host.refs > 0).sum()
    reserve([70, 5, 0, 1, 1, 200, 0, 1, 1])
    pages.compact()
    host.compact()
    host.same(T, pages)


@pytest.mark.parametrize("seed", range(6))
def test_random_calls(cuda, seed):
    import torch as T
    rng = np.random.default_rng(seed)
    S, wide, nb = int(rng.integers(1, 40)), int(rng.integers(1, 12)), int(rng.integers(3, 260))
    host = Host(rng, S, wide, nb, 2, 2, 64)
    pages = host.device(T)
    lens = np.zeros(S, np.int64)
    for _ in range(25):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            new = np.where(rng.random(S) < 0.6, rng.integers(1, 90, S), 0)
            back = np.where(rng.random(S) < 0.1, rng.integers(0, 70, S), 0)
            after = np.minimum(np.maximum(lens - back, 0) + new, wide * BLOCK)
            new = np.where(new > 0, np.minimum(new, after), 0)
            lens = np.where(new > 0, after, lens)
            if new.sum() == 0:
                continue
            host.reserve(new.tolist(), lens.tolist())
            pages.reserve(batch_of(new.tolist(), lens.tolist()))
        elif what == "fork":
            n = int(rng.integers(1, S + 1))
            p, c = rng.integers(-1, S + 1, n), rng.integers(-1, S + 1, n)
            k = rng.integers(-3, wide * BLOCK + 9, n)
            was = lens.copy()
            seen = set()
            for a, b, m in zip(p, c, k):
                if 0 <= b < S and b not in seen:
                    seen.add(b)
                    if 0 <= a < S and a != b:
                        lens[b] = min(max(m, 0), was[a])
            host.fork(p.tolist(), c.tolist(), k.tolist())
            pages.fork(i32(T, p.tolist()), i32(T, c.tolist()), i32(T, k.tolist()))
        elif what == "free":
            q = rng.integers(-1, S + 1, int(rng.integers(1, S + 1)))
            lens[[s for s in q if 0 <= s < S]] = 0
            host.free(q.tolist())
            pages.free(i32(T, q.tolist()))
        else:
            most = None if rng.random() < 0.5 else int(rng.integers(0, 6))
            host.compact(most)
            pages.compact(most)
        host.same(T, pages)


@pytest.mark.parametrize("n_blocks", [1, 15, 16, 17, 4099, 16384, 16385, 70001])
def test_many_blocks(cuda, n_blocks):
    """Pools around the rounds in which blocks are looked through: half of them live, scattered."""
    import torch as T
    rng = np.random.default_rng(n_blocks)
    wide = max(1, n_blocks // 50)
    host = Host(rng, 50, wide, n_blocks, 1, 1, 64)
    host.layers[0]["k"][:] = (np.arange(n_blocks) % 251).astype(np.uint8)[:, None, None, None, None]
    half = rng.permutation(n_blocks)[:n_blocks // 2]
    host.table.reshape(-1)[rng.permutation(50 * wide)[:len(half)]] = half[:50 * wide]
    host.refs[:] = np.bincount(host.table[host.table >= 0], minlength=n_blocks)
    pages = host.device(T)
    for most in (0, n_blocks // 10, None):
        host.compact(most)
        pages.compact(most)
        host.same(T, pages)
    new = [BLOCK * wide] * 50
    host.reserve(new, new)
    pages.reserve(batch_of(new, new))
    host.same(T, pages)


def test_many_sequences(cuda):
    import torch as T
    rng = np.random.default_rng(1)
    S = 2500
    host = Host(rng, S, 3, 6000, 1, 1, 64)
    pages = host.device(T)
    new = rng.integers(0, 150, S).tolist()
    host.reserve(new, new)
    pages.reserve(batch_of(new, new))
    host.same(T, pages)
    p, c = rng.permutation(S).tolist(), rng.permutation(S).tolist()
    k = [new[a] for a in p]
    host.fork(p, c, k)
    pages.fork(i32(T, p), i32(T, c), i32(T, k))
    host.same(T, pages)


@pytest.mark.parametrize("wide", [250, 700])
def test_forks_of_long_rows(cuda, wide):
    """Rows that the plan's thread block makes itself, and more of them than it does."""
    import torch as T
    rng = np.random.default_rng(wide)
    S, nb = 60, 9000
    lens = [int(n) for n in rng.integers(1, 130 * BLOCK, S)]
    host = Host(rng, S, wide, nb, 1, 1, 64).fill(rng, lens)
    host.layers[0]["v"][:] = (np.arange(nb) % 253).astype(np.uint8)[:, None, None, None]
    pages = host.device(T)
    for n in (3, 60, 25):
        p, c = rng.integers(0, S, n).tolist(), rng.permutation(S)[:n].tolist()
        k = [int(rng.integers(0, lens[a] + 1)) for a in p]
        host.fork(p, c, k)
        pages.fork(i32(T, p), i32(T, c), i32(T, k))
        host.same(T, pages)
        was = list(lens)
        for a, b, m in zip(p, c, k):
            lens[b] = m if a != b else was[b]


def test_too_few_blocks(cuda):
    """What is left without a block is -1, the word says so once, and the others are whole."""
    import torch as T
    rng = np.random.default_rng(2)
    host = Host(rng, 4, 4, 6, 1, 2, 64)
    pages = host.device(T)
    for new, lens in (([100, 64, 1, 0], [100, 64, 1, 0]), ([64, 64, 64, 0], [164, 128, 65, 0])):
        host.reserve(new, lens)
        pages.reserve(batch_of(new, lens))
    assert (host.table >= 0).sum() == 6 and host.error == 1
    host.same(T, pages)
    host.fork([0, 0], [3, 2], [90, 70])
    pages.fork(i32(T, [0, 0]), i32(T, [3, 2]), i32(T, [90, 70]))
    assert host.error == 1
    host.same(T, pages)
    host.free([0])
    pages.free(i32(T, [0]))
    host.same(T, pages)                                                            # (the word was zeroed)


def test_table_with_numbers_outside_the_cache(cuda):
    import torch as T
    rng = np.random.default_rng(3)
    host = Host(rng, 3, 4, 12, 1, 1, 64).fill(rng, [200, 64, 0])
    host.table[1, 1], host.table[1, 2], host.table[2, 0] = 12, -5, 1 << 30
    pages = host.device(T)
    for call in ("fork", "reserve", "compact", "free"):
        if call == "fork":
            host.fork([1, 0], [2, 1], [190, 130])
            pages.fork(i32(T, [1, 0]), i32(T, [2, 1]), i32(T, [190, 130]))
        elif call == "reserve":
            host.reserve([1, 100, 10], [201, 230, 200])
            pages.reserve(batch_of([1, 100, 10], [201, 230, 200]))
        elif call == "compact":
            host.compact()
            pages.compact()
        else:
            host.free([1, 2])
            pages.free(i32(T, [1, 2]))
        host.same(T, pages)


def test_copy(cuda):
    import torch as T
    rng = np.random.default_rng(4)
    for layers, kv, dim in ((1, 1, 64), (4, 3, 192), (2, 8, 128)):
        host = Host(rng, 1, 1, 40, layers, kv, dim)
        pages = host.device(T)
        order = rng.permutation(40)
        src, dst = order[:17].tolist(), order[17:34].tolist()
        host.move(list(zip(src, dst)))
        pages.copy(i32(T, src + [-1, 40, 3]), i32(T, dst + [order[35], order[36], 1 << 20]))       # (no such blocks: passed over)
        host.same(T, pages)
        pages.copy(i32(T, []), i32(T, []))


def test_counts_made_from_the_table(cuda):
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(5)
    host = Host(rng, 3, 4, 12).fill(rng, [200, 64, 0])
    host.table[2] = host.table[0]
    host.refs[host.table[0]] = 2
    pages = host.device(T)
    assert T.equal(api.KvPages(pages.caches).refs, pages.refs)


def test_captured_steps(cuda):
    """Steps of decode with their blocks handed out in one graph, replayed: each replay does what the table and the lengths then ask for."""
    import torch as T
    from project_maya_b200 import api
    rng = np.random.default_rng(6)
    host = Host(rng, 5, 6, 40, 2, 1, 64).fill(rng, [60, 64, 1, 100, 0])
    pages = host.device(T)
    host.fork([3], [4], [70])
    pages.fork(i32(T, [3]), i32(T, [4]), i32(T, [70]))
    lens = [60, 64, 1, 100, 70]
    kv_len, start = i32(T, lens), T.arange(6, dtype=T.int32, device="cuda")
    batch = api.AttnBatch(start, kv_len, 5, 1, 6 * BLOCK)
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        kv_len.add_(1)
        pages.reserve(batch)
    for _ in range(70):
        lens = [n + 1 for n in lens]
        host.reserve([1] * 5, lens)
        g.replay()
    T.cuda.synchronize()
    host.same(T, pages)
    assert kv_len.tolist() == lens


def test_forked_sequences_attend_as_if_they_had_their_own_blocks(cuda):
    """Append, fork, reserve, append, attend: beside the same sequences in caches of their own, bit for bit."""
    import torch as T
    from project_maya_b200 import api
    T.manual_seed(7)
    dim, kv, n_q = 64, 2, 4
    table = T.full((3, 5), -1, dtype=T.int32, device="cuda")
    cache = api.KvCache.empty(16, kv, dim, table)
    own = api.KvCache.empty(16, kv, dim, T.arange(15, dtype=T.int32, device="cuda").view(3, 5))
    pages = api.KvPages([cache])
    attn, plain = api.KvAttention(cache, n_q), api.KvAttention(own, n_q)
    rope = api.Rope()

    def step(new, lens, reserve=True):
        b = batch_of(new, lens)
        n = sum(new)
        q, k, v = T.randn((n, n_q, dim), device="cuda"), T.randn((n, kv, dim), device="cuda"), T.randn((n, kv, dim), device="cuda")
        if reserve:
            pages.reserve(b)
        attn.append(b, q, k, v, rope)
        plain.append(b, q, k, v, rope)
        assert T.equal(attn.forward(b, q), plain.forward(b, q))

    def join():                                                                    # the children's prefixes in the cache of their own
        own_blocks, blocks = own.table.view(-1).long(), cache.table.view(-1)
        for o, c in zip(own_blocks.tolist(), blocks.tolist()):
            if c >= 0:
                for n in PARTS:
                    getattr(own, n)[o] = getattr(cache, n)[c]

    step([100, 0, 0], [100, 0, 0])
    pages.fork(i32(T, [0, 0]), i32(T, [1, 2]), i32(T, [100, 64]))
    join()
    for i in range(40):
        step([1, 1, 1], [101 + i, 101 + i, 65 + i])
    pages.fork(i32(T, [2, 1]), i32(T, [0, 2]), i32(T, [90, 140]))
    join()
    step([3, 1, 2], [93, 141, 142])
    step([1, 0, 1], [20, 0, 130])                                                   # both taken back, sequence 0 into a block that it shares
    step([1, 1, 1], [21, 142, 131])
    pages.free(i32(T, [1]))
    pages.compact()
    step([1, 0, 1], [22, 0, 132])
    assert pages.error() == 0 and attn.error() == 0


@pytest.mark.parametrize("wide,n", [(96, 32), (96, 33), (97, 32), (5000, 1)])
def test_forks_on_both_sides_of_the_choice(cuda, wide, n):
    """The most rows and blocks a row that the plan's thread block takes, one more of each, and a single long row."""
    import torch as T
    rng = np.random.default_rng(wide + n)
    S, nb = 40, 6000
    lens = [int(v) for v in rng.integers(1, min(wide, 100) * BLOCK, S)]
    if n == 1:
        lens[7] = 4000 * BLOCK + 5
    host = Host(rng, S, wide, nb + 4000 * (n == 1), 1, 1, 64).fill(rng, lens)
    pages = host.device(T)
    p, c = ([7], [3]) if n == 1 else (rng.integers(0, S, n).tolist(), rng.permutation(S)[:n].tolist())
    k = [lens[a] - 2 if lens[a] > 2 else lens[a] for a in p]
    host.fork(p, c, k)
    pages.fork(i32(T, p), i32(T, c), i32(T, k))
    host.same(T, pages)


def test_a_shortage_loses_what_stood_in_a_block_that_was_to_be_replaced(cuda):
    """Two sequences share the block that both go on in, and none is free: both entries are -1, the tokens in them are lost to both, a later reserve gives blocks and not
    their tokens.  Who holds other blocks keeps them; prefilled from the start, the two are whole again."""
    import torch as T
    rng = np.random.default_rng(8)
    host = Host(rng, 3, 3, 4, 1, 1, 64).fill(rng, [100, 0, 128])
    pages = host.device(T)
    host.fork([0], [1], [64])
    pages.fork(i32(T, [0]), i32(T, [1]), i32(T, [64]))
    host.table[1, 1] = host.table[0, 1]                                            # (shared by the caller)
    host.refs[host.table[0, 1]] = 2
    pages.table.copy_(T.from_numpy(host.table))
    pages.refs.copy_(T.from_numpy(host.refs))
    kept = host.table[2].copy()
    host.reserve([1, 1, 0], [101, 101, 0])
    pages.reserve(batch_of([1, 1, 0], [101, 101, 0]))
    assert host.error == 1 and (host.table[:2, 1] == -1).all() and (host.table[2] == kept).all()
    host.same(T, pages)
    host.free([0, 1])
    pages.free(i32(T, [0, 1]))
    host.reserve([101, 0, 0], [101, 0, 0])
    pages.reserve(batch_of([101, 0, 0], [101, 0, 0]))
    assert host.error == 0 and (host.table[0, :2] >= 0).all() and (host.table[2] == kept).all()
    host.same(T, pages)
