"""What a decoder layer that serves many requests needs between its products and around its cache, as cases that can be timed.

  norm     rows of the residual stream plus what a half of the layer adds to them, their RMS norm times a weight, and the normed rows in 8 bits
           with scales for the product behind it (q8_1 blocks or the prompt path's image); the 8-bit rows read back as the values they stand for
  route    experts of each token: softmax or sigmoid scores, a bias that only chooses, groups of neighbouring experts of which the best are
           kept, the k best experts of these, their weights
  adapt    low-rank adapters beside a projection that all requests share: y[t] + scale[i] * B[i] (A[i] x[t]) with i = idx[t], -1: none
  fork     beams go on from other beams: full blocks of the cache are shared, the block in the middle of which a beam stands is copied; then room
           for each beam's next token
  turn     some sequences leave, what is left moves to the front of the cache's blocks, and as many new sequences get room
  copy     blocks copied to others, in all layers

Blocks: refs[b] tables hold block b, 0: it is free; whoever needs blocks gets the free ones of the lowest numbers, in the order of asking.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64
EPS = 1e-6
LEAST = 2.0 ** -14                                   # what a sum of weights is divided by at least
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _norm(rows, n, act, form, add=True, **more):
    return dict(op="norm", rows=rows, n=n, act=act, form=form, add=add, **more)


def _route(tokens, experts, k, groups, keep, sigmoid, top2, bias, **more):
    return dict(op="route", tokens=tokens, experts=experts, k=k, groups=groups, keep=keep, sigmoid=sigmoid, top2=top2, bias=bias, **more)


def _adapt(tokens, n_in, n_out, rank, adapters, act, weights, runs, **more):
    """runs: the adapter changes every so many tokens (1: each token has its own)."""
    return dict(op="adapt", tokens=tokens, n_in=n_in, n_out=n_out, rank=rank, adapters=adapters, act=act, weights=weights, runs=runs, **more)


def _pages(op, seqs, length, some, layers, kv, dim, **more):
    """some: beams of a group (fork), sequences that leave (turn), blocks that are copied (copy)."""
    return dict(op=op, seqs=seqs, len=length, some=some, layers=layers, kv=kv, dim=dim, **more)


def listed():
    return [
        # one token in front of its projections: the residual stream, what attention added, q8_1 blocks for the GEMV
        _norm(1, 6144, "f32", "q8_1", name="norm_token"),
        # a window of 13 tokens in front of the router: bf16 rows, the normed rows in f32
        _norm(13, 7168, "bf16", "rows", name="norm_window"),
        # a prompt chunk in front of the prompt path's product
        _norm(4096, 6144, "f32", "mmq", name="norm_prompt"),
        # one token over 8 groups of 32 experts, sigmoid scores and a bias
        _route(1, 256, 8, 8, 4, True, True, True, name="route_token"),
        # a decode batch over 160 experts, softmax scores
        _route(61, 160, 6, 8, 3, False, False, False, name="route_batch"),
        # two prompt chunks
        _route(8192, 256, 8, 8, 4, True, True, True, name="route_prompt"),
        # one token with its adapter beside the query, key and value rows
        _adapt(1, 4096, 6144, 16, 8, "f32", "bf16", 1, name="adapt_token"),
        # a decode batch of 64 requests that use 24 adapters
        _adapt(64, 4096, 6144, 16, 24, "f32", "f16", 1, name="adapt_batch"),
        # prompts of requests with adapters of their own, one of four without
        _adapt(4096, 4096, 6144, 64, 3, "f32", "bf16", 1100, name="adapt_prompt"),
        # eight groups of four beams at some 1500 tokens
        _pages("fork", 32, 1500, 4, 2, 8, 128, name="pages_fork"),
        # 48 requests, four of which leave
        _pages("turn", 48, 1500, 4, 2, 8, 128, name="pages_turn"),
        # 500 blocks of four layers
        _pages("copy", 48, 1500, 500, 4, 8, 128, name="pages_copy"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        at = most.setdefault(c["op"], [0, 0])
        at[0], at[1] = max(at[0], w["bytes"]), max(at[1], w["flops"])
    while True:
        op = rng.choice(("norm", "route", "adapt", "adapt", "fork", "turn", "copy"))
        if op == "norm":
            c = _norm(_log_int(rng, 1, 4096), 32 * _log_int(rng, 16, 512), rng.choice(("f32", "bf16")), rng.choice(("q8_1", "mmq", "rows")),
                      rng.random() < 0.7)
        elif op == "route":
            groups = rng.choice((1, 2, 4, 5, 8, 16))
            keep = rng.randint(1, groups)
            experts = groups * _log_int(rng, 4, 512 // groups)
            k = rng.randint(1, min(16, keep * (experts // groups)))
            c = _route(_log_int(rng, 1, 8192), experts, k, groups, keep, rng.random() < 0.6, rng.random() < 0.6, rng.random() < 0.6)
        elif op == "adapt":
            tokens = _log_int(rng, 1, 4096)
            c = _adapt(tokens, 32 * _log_int(rng, 16, 224), _log_int(rng, 500, 7168), rng.choice((4, 8, 16, 16, 24, 32, 64)),
                       rng.randint(1, 3) if tokens > 512 else _log_int(rng, 1, 32), rng.choice(("f32", "f32", "bf16")), rng.choice(("bf16", "f16")),
                       rng.choice((1, 1, _log_int(rng, 1, tokens))))
        else:
            seqs = 4 * rng.randint(1, 12)
            some = rng.choice((2, 4)) if op != "copy" else _log_int(rng, 1, 500)
            c = _pages(op, seqs, _log_int(rng, 70, 3000), some, rng.randint(1, 4), rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 192)))
        w = work(c)
        if w["bytes"] > most[op][0] or w["flops"] > most[op][1]:
            continue
        if op == "copy" and 2 * c["some"] > _pool(c):
            continue
        return c


# ---------------------------------------------------------------- what a case holds
def _lengths(c):
    """Tokens of every sequence: alike where sequences take one another's place, else ragged."""
    if c["op"] == "turn":
        return [c["len"]] * c["seqs"]
    return [max(1, round(c["len"] * (1 - 0.3 * (0.618034 * i % 1)))) for i in range(c["seqs"])]


def _blocks(n):
    return -(-n // BLOCK)


def _wide(c):
    return _blocks(c["len"]) + 2


def _pool(c):
    need = sum(_blocks(n) for n in _lengths(c))
    return need + (3 * c["seqs"] + 5 if c["op"] != "copy" else need // 4)


def _adapter_of(c):
    """The adapter of every token: runs of tokens, one run in four (where there are runs) without any."""
    run, n = c["runs"], c["adapters"]
    out = []
    for t in range(c["tokens"]):
        i = t // run
        out.append(-1 if i % 4 == 2 else (i * 7 + 1) % n if run == 1 else i % n)
    return out


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(g, *shape):
    return torch.randint(1, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    c, g, dev = case, _gen(seed), torch.device("cuda")
    randn = lambda *shape: torch.randn(shape, generator=g, device=dev)                # noqa: E731
    st = dict(case=dict(c))
    if c["op"] == "norm":
        T, n = c["rows"], c["n"]
        # a stream whose rows differ in size, with a few large columns, as layers in the middle of a model see it
        st["h"] = (randn(T, n) * (0.5 + torch.rand((T, 1), generator=g, device=dev)) * (1 + 9 * (torch.rand(n, generator=g, device=dev) < 0.004))).to(TYPES[c["act"]])
        st["add"] = (0.3 * randn(T, n)).to(TYPES[c["act"]]) if c["add"] else None
        st["w"] = 1 + 0.1 * randn(n)
        st["h_out"] = torch.empty_like(st["h"]) if c["add"] else None
    elif c["op"] == "route":
        E = c["experts"]
        st["logits"] = 1.5 * randn(c["tokens"], E) + 0.5 * randn(E)
        st["bias"] = 0.05 * randn(E) if c["bias"] else None
    elif c["op"] == "adapt":
        n, r, act, wt = c["adapters"], c["rank"], TYPES[c["act"]], TYPES[c["weights"]]
        st["x"] = randn(c["tokens"], c["n_in"]).to(act)
        st["y"] = randn(c["tokens"], c["n_out"])
        st["a"] = (randn(n, r, c["n_in"]) / c["n_in"] ** 0.5).to(wt)
        st["b"] = (randn(n, c["n_out"], r) / r ** 0.5).to(wt)
        st["scale"] = 0.25 + torch.rand(n, generator=g, device=dev)
        turn = torch.randperm(n, generator=g, device=dev, dtype=torch.int32)
        of = torch.tensor(_adapter_of(c), dtype=torch.int32, device=dev)
        st["idx"] = torch.where(of < 0, of, turn[of.clamp(min=0).long()])
        st["out"] = torch.empty_like(st["y"])
    else:
        L, KV, D, nb, S, wide, lens = c["layers"], c["kv"], c["dim"], _pool(c), c["seqs"], _wide(c), _lengths(c)
        st["k"], st["v"] = _codes(g, L, nb, KV, D // 64, BLOCK, 64), _codes(g, L, nb, KV, D, BLOCK)
        st["k_scale"], st["v_scale"] = (0.02 * (1 + torch.rand((L, nb, KV), generator=g, device=dev)) for _ in range(2))
        st["k_sum"] = torch.randint(-8000, 8000, (L, nb, KV, D), generator=g, device=dev, dtype=torch.int16)
        order = torch.randperm(nb, generator=g, device=dev, dtype=torch.int32)        # blocks as an allocator that has run for a while holds them
        table = torch.full((S, wide), -1, dtype=torch.int32, device=dev)
        need, at = [_blocks(n) for n in lens], 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        st["table"], st["refs"] = table, torch.zeros(nb, dtype=torch.int32, device=dev)
        st["refs"][order[:at].long()] = 1
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)                # noqa: E731
        if c["op"] == "fork":
            pick = torch.rand(S, generator=g, device=dev) * c["some"]                 # each beam goes on from one of its group's
            st["children"] = torch.arange(S, dtype=torch.int32, device=dev)
            st["parents"] = (st["children"] // c["some"]) * c["some"] + pick.int()
            st["lens"] = i32(lens).view(-1, c["some"]).amin(1).repeat_interleave(c["some"])       # beams of a group are equally long
            st["start"], st["kv_len"] = torch.arange(S + 1, dtype=torch.int32, device=dev), st["lens"] + 1
        elif c["op"] == "turn":
            m, n = c["some"], c["len"]
            rounds = [[(m * r + i) % S for i in range(m)] for r in range(S // math.gcd(S, m))]
            st["leave"] = [i32(q) for q in rounds]
            st["start"] = [i32([n * sum(j in q for j in range(s)) for s in range(S + 1)]) for q in rounds]
            st["kv_len"] = [i32([n if s in q else 0 for s in range(S)]) for q in rounds]
            st["round"] = 0
        else:
            both = torch.randperm(nb, generator=g, device=dev, dtype=torch.int32)
            st["src"], st["dst"] = both[:c["some"]].contiguous(), both[c["some"]:2 * c["some"]].contiguous()
    return st


# ---------------------------------------------------------------- the plain forms
def _away(x):
    """Rounded to whole numbers, halves away from zero."""
    return torch.copysign(torch.floor(x.abs() + 0.5), x)


def _plain_norm(st):
    c = st["case"]
    t = st["h"].float()
    if c["add"]:
        t = t + st["add"].float()
        st["h_out"].copy_(t)
    x = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * st["w"]
    if c["form"] == "rows":
        return {"x": x, "h": st["h_out"]}
    v = x.view(c["rows"], -1, 32)
    amax = v.abs().amax(-1, keepdim=True)
    if c["form"] == "q8_1":
        d = (amax / 127).clamp(max=65504.0)
        q = torch.where(amax > 0, _away(v / d), 0.0)
        d = d.half().float()
    else:
        inv = 127 / amax
        q = torch.where(amax > 0, _away(v * inv), 0.0)
        d = torch.where(amax > 0, 1 / inv, 0.0).clamp(max=65504.0).half().float()
    q = d * q.clamp(-127, 127)
    if c["form"] == "mmq":
        q = q.half().float()
    return {"values": q.view(c["rows"], -1).bfloat16(), "sums": v.sum(-1).half(), "h": st["h_out"]}


def _plain_route(st):
    c = st["case"]
    T, E, G = c["tokens"], c["experts"], c["groups"]
    l = st["logits"].double()                                                         # scores next to one another decide the choice
    if c["sigmoid"]:
        s = 1 / (1 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    by = s if st["bias"] is None else s + st["bias"].double()
    if c["keep"] < G:
        g = by.view(T, G, -1)
        best = torch.sort(g, dim=-1, descending=True).values
        best = best[..., :2].sum(-1) if c["top2"] else best[..., 0]
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
        out = torch.ones((T, G), dtype=torch.bool, device=l.device).scatter_(1, kept, False)
        by = g.masked_fill(out[..., None], -math.inf).view(T, E)
    ids = torch.sort(by, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = s.gather(1, ids)
    w = 2.5 * w / w.sum(-1, keepdim=True).clamp(min=LEAST)
    return {"ids": ids.int(), "weights": w.float()}


def _plain_adapt(st):
    c = st["case"]
    T, n, r = c["tokens"], c["adapters"], c["rank"]
    # every adapter's product, of which a token keeps its own adapter's
    z = torch.matmul(st["x"].float(), st["a"].float().view(n * r, -1).t()).view(T, n, r)
    mine = st["idx"][:, None] == torch.arange(n, device=z.device)
    z = torch.where(mine[..., None], z * st["scale"][:, None], 0.0).view(T, n * r)
    st["out"].copy_(st["y"] + torch.matmul(z, st["b"].float().transpose(0, 1).reshape(c["n_out"], n * r).t()))
    return st["out"]


CACHE = ("k", "v", "k_scale", "v_scale", "k_sum")


def _plain_move(st, src, dst):
    st["k"][:, dst], st["v"][:, dst], st["k_sum"][:, dst] = st["k"][:, src], st["v"][:, src], st["k_sum"][:, src]
    st["k_scale"][:, dst], st["v_scale"][:, dst] = st["k_scale"][:, src], st["v_scale"][:, src]


def _count(refs, blocks, valid, by):
    refs.scatter_add_(0, torch.where(valid, blocks, 0).long().flatten(), torch.where(valid, by, 0).int().flatten())


def _plain_fork(st):
    table, refs = st["table"], st["refs"]
    p, ch, n = st["parents"].long(), st["children"].long(), st["lens"].long()
    moved = p != ch
    full, part = n // BLOCK, (n % BLOCK > 0) & moved
    free = torch.sort((refs > 0).int(), stable=True).indices.int()
    new = free[(part.cumsum(0) - 1).clamp(min=0)]
    col = torch.arange(table.shape[1], device=table.device)
    rows, old = table[p], table[ch]
    shared = (col < full[:, None]) & moved[:, None]
    at = (col == full[:, None]) & part[:, None]
    partial = rows.gather(1, full[:, None]).squeeze(1)
    row = torch.where(shared, rows, torch.where(at, new[:, None], -1))
    _count(refs, rows, shared & (rows >= 0), 1)
    _count(refs, old, (old >= 0) & moved[:, None], -1)
    _count(refs, new, part, 1)
    table[ch] = torch.where(moved[:, None], row, old)
    _plain_move(st, torch.where(part, partial, refs.numel() - 1).long(), torch.where(part, new, refs.numel() - 1).long())


def _plain_reserve(st, start, kv_len):
    table, refs = st["table"], st["refs"]
    new = (start[1:] - start[:-1]).long()
    first, last = (kv_len - new) // BLOCK, (kv_len - 1) // BLOCK
    col = torch.arange(table.shape[1], device=table.device)
    want = (new[:, None] > 0) & (col >= first[:, None]) & (col <= last[:, None])
    want &= (table < 0) | (refs[table.clamp(min=0).long()] > 1)                       # (in these cases no shared block is written to)
    free = torch.sort((refs > 0).int(), stable=True).indices.int()
    got = free[(want.flatten().cumsum(0) - 1).clamp(min=0, max=refs.numel() - 1)].view_as(table)
    _count(refs, got, want, 1)
    table.copy_(torch.where(want, got, table))


def _plain_free(st, seqs):
    old = st["table"][seqs.long()]
    _count(st["refs"], old, old >= 0, -1)
    st["table"][seqs.long()] = -1


def _plain_compact(st, most):
    table, refs = st["table"], st["refs"]
    nb = refs.numel()
    at = torch.arange(nb, device=refs.device)
    live = refs > 0
    n = live.sum()
    hole, tail = ~live & (at < n), live & (at >= n)
    dst = torch.sort((~hole).int(), stable=True).indices[:most]
    src = torch.sort((~tail).int(), stable=True).indices[:most]
    real = torch.arange(most, device=refs.device) < hole.sum()
    to = torch.cat((at, at[:1]))
    to[torch.where(real, src, nb)] = dst
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    counts = torch.cat((refs, refs[:1]))
    counts[torch.where(real, dst, nb)] = refs[src]
    counts[torch.where(real, src, nb)] = 0
    refs.copy_(counts[:nb])
    last = torch.full_like(src, nb - 1)                                               # (no block moves there: copied onto itself)
    _plain_move(st, torch.where(real, src, last), torch.where(real, dst, last))


def _pages_out(st):
    return {name: st[name] for name in CACHE} | {"table": st["table"], "refs": st["refs"]}


def _plain_pages(st):
    c = st["case"]
    if c["op"] == "copy":
        _plain_move(st, st["src"].long(), st["dst"].long())
    elif c["op"] == "fork":
        _plain_fork(st)
        _plain_reserve(st, st["start"], st["kv_len"])
    else:
        r = st["round"]
        st["round"] = (r + 1) % len(st["leave"])
        _plain_free(st, st["leave"][r])
        _plain_compact(st, c["some"] * _blocks(c["len"]))
        _plain_reserve(st, st["start"][r], st["kv_len"][r])
    return _pages_out(st)


# ---------------------------------------------------------------- one pass
def _own_norm(st):
    from project_maya_b200 import api
    c = st["case"]
    if c["form"] == "rows":
        if "x" not in st:
            st["x"] = torch.empty((c["rows"], c["n"]), dtype=torch.float32, device=st["h"].device)
        api.rms_q8(st["h"], st["add"], st["w"], EPS, image=None, h_out=st["h_out"], x=st["x"])
        return {"x": st["x"], "h": st["h_out"]}
    image = api.XQ_Q8_1 if c["form"] == "q8_1" else api.XQ_MMQ
    xq = api.rms_q8(st["h"], st["add"], st["w"], EPS, image=image, h_out=st["h_out"])
    values, sums = api.q8_read(xq, c["rows"], c["n"], image)
    return {"values": values, "sums": sums, "h": st["h_out"]}


def _own_route(st):
    from project_maya_b200 import api
    c = st["case"]
    ids, weights = api.router_groups(st["logits"], c["k"], n_group=c["groups"], n_keep=c["keep"], bias=st["bias"], sigmoid=c["sigmoid"],
                                     top2=c["top2"], w_scale=2.5)
    return {"ids": ids, "weights": weights}


def _own_adapt(st):
    from project_maya_b200 import api
    if "adapters" not in st:
        st["adapters"] = api.LoraAdapters(st["a"], st["b"], st["scale"], max_tokens=st["case"]["tokens"])
    return st["adapters"].forward(st["x"], st["idx"], st["y"], out=st["out"])


def _own_pages(st):
    from project_maya_b200 import api
    c = st["case"]
    if "pages" not in st:
        st["pages"] = api.KvPages([api.KvCache(*(st[name][i] for name in CACHE[:4]), st["table"], k_sum=st["k_sum"][i]) for i in range(c["layers"])],
                                  st["refs"])
        if c["op"] == "fork":
            st["batches"] = [api.AttnBatch(st["start"], st["kv_len"], c["seqs"], 1, c["len"] + 1)]
        elif c["op"] == "turn":
            st["batches"] = [api.AttnBatch(a, b, c["some"] * c["len"], c["len"], c["len"]) for a, b in zip(st["start"], st["kv_len"])]
    pages = st["pages"]
    if c["op"] == "copy":
        pages.copy(st["src"], st["dst"])
    elif c["op"] == "fork":
        pages.fork(st["parents"], st["children"], st["lens"])
        pages.reserve(st["batches"][0])
    else:
        r = st["round"]
        st["round"] = (r + 1) % len(st["leave"])
        pages.free(st["leave"][r])
        pages.compact(c["some"] * _blocks(c["len"]))
        pages.reserve(st["batches"][r])
    return _pages_out(st)


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_norm if op == "norm" else _own_route if op == "route" else _own_adapt if op == "adapt" else _own_pages)(state)
    return (_plain_norm if op == "norm" else _plain_route if op == "route" else _plain_adapt if op == "adapt" else _plain_pages)(state)


def work(case):
    c = case
    if c["op"] == "norm":
        es = 4 if c["act"] == "f32" else 2
        N = c["rows"] * c["n"]
        out = {"q8_1": 2 + 36 / 32 + 2 / 32, "mmq": 2 + 2 + 2 / 32 + 2 / 32, "rows": 4}[c["form"]]
        return {"bytes": N * (es * (3 if c["add"] else 1) + out) + 4 * c["n"], "flops": 8 * N}
    if c["op"] == "route":
        n = c["tokens"] * c["experts"]
        return {"bytes": 4 * n + 8 * c["tokens"] * c["k"] + (4 * c["experts"] if c["bias"] else 0), "flops": 40 * n}
    if c["op"] == "adapt":
        of = _adapter_of(c)
        used, live = len(set(of) - {-1}), sum(i >= 0 for i in of)
        es = 4 if c["act"] == "f32" else 2
        return {"bytes": live * c["n_in"] * es + 8 * c["tokens"] * c["n_out"] + 2 * used * c["rank"] * (c["n_in"] + c["n_out"]),
                "flops": 2 * live * c["rank"] * (c["n_in"] + c["n_out"])}
    # blocks that move: each read and written
    block = c["layers"] * c["kv"] * (2 * BLOCK * c["dim"] + 2 * c["dim"] + 8)
    moved = c["some"] if c["op"] == "copy" else c["some"] * _blocks(c["len"]) if c["op"] == "turn" else c["seqs"] * (c["some"] - 1) // c["some"]
    index = 4 * c["seqs"] * _wide(c) * 2 + 4 * _pool(c)
    return {"bytes": 2 * moved * block + (index if c["op"] != "copy" else 8 * moved), "flops": 0}


# ---------------------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    c = case
    if c["op"] in ("fork", "turn", "copy"):                                           # whole numbers and moved bytes: nothing is rounded
        return None
    st = prepare(c, seed)
    if c["op"] == "norm":
        t = st["h"].double() + (st["add"].double() if c["add"] else 0)
        h = t if c["add"] else None
        x = t / torch.sqrt(torch.linalg.vector_norm(t, dim=1, keepdim=True) ** 2 / c["n"] + EPS) * st["w"].double()
        if c["form"] == "rows":
            return {"x": x, "h": h}
        b = x.unflatten(1, (-1, 32))
        step = b.abs().max(-1, keepdim=True).values / 127
        values = torch.sign(b) * torch.floor(b.abs() / step + 0.5) * step
        return {"values": torch.nan_to_num(values).flatten(1), "sums": b.sum(-1), "h": h}
    if c["op"] == "route":
        l = st["logits"].double()
        p = torch.sigmoid(l) if c["sigmoid"] else torch.softmax(l, -1)
        score = p if st["bias"] is None else p + st["bias"].double()
        per = c["experts"] // c["groups"]
        group = torch.topk(score.unflatten(1, (c["groups"], per)), min(per, 2 if c["top2"] else 1), dim=-1).values.sum(-1)
        inside = torch.zeros_like(group).scatter_(1, torch.topk(group, c["keep"], dim=-1).indices, 1.0).repeat_interleave(per, 1) > 0
        chosen = torch.topk(torch.where(inside, score, -math.inf), c["k"], dim=-1).indices
        w = torch.take_along_dim(p, chosen, 1)
        return {"ids": None, "weights": w / torch.maximum(w.sum(1, keepdim=True), torch.tensor(LEAST, dtype=torch.float64, device=w.device)) * 2.5}
    out = st["y"].double()
    for i in range(c["adapters"]):
        rows = torch.nonzero(st["idx"] == i).flatten()
        z = st["x"][rows].double() @ st["a"][i].double().T
        out[rows] += st["scale"][i].double() * (z @ st["b"][i].double().T)
    return out
