"""The attention half of a decoder layer over a paged cache of 8-bit keys and values, as cases that can be timed.

  append   queries and keys normalised per head and rotated by their positions, keys and values rounded into the cache's blocks; then
           the blocks that were touched read back as the values they stand for
  attn     attention of the new tokens over their sequences in the cache (causal; `window` > 0: over the last `window` positions)
  select   the blocks each new token reads, for each group of heads: the first and the last ones, and those whose summed keys score highest
  sparse   attention of the new tokens over selected blocks alone

The cache: blocks of 64 tokens; a block and key/value head hold 64 * dim codes (value / scale + 128, one byte) and one f32 scale for the
keys and one for the values.  Keys [block][head][dim / 64][token][64], values [block][head][dim][token]; k_sum [block][head][dim] int16
is the sum of the keys' codes (less 128) over the block's tokens.  Sequence s holds its tokens 64 b .. 64 b + 63 in block table[s][b].
New tokens are packed: those of sequence s are rows start[s] .. start[s + 1] - 1, the last of its kv_len[s] tokens.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
INV127 = 1.0 / 127.0


def _case(op, seqs, new, length, heads, kv, dim, act, **more):
    c = dict(op=op, seqs=seqs, new=new, len=length, heads=heads, kv=kv, dim=dim, act=act, ragged=False, window=0, sel=0, first=1,
             last=2, rot=dim, pairs=False)
    c.update(more)
    return c


def listed():
    return [
        # the smallest calls: one token of one chat, f32 activations as the GEMVs in front leave them - launches and latency
        dict(_case("append", 1, 1, 1000, 32, 8, 128, "f32"), name="append_token"),
        # a decode batch of 64 requests at ragged lengths
        dict(_case("append", 64, 1, 8192, 64, 8, 128, "bf16", ragged=True), name="append_batch"),
        # three prompts chunks of ragged lengths, behind what their sequences hold already; 48 heads, half of each rotated in pairs
        dict(_case("append", 3, 2500, 4001, 48, 8, 128, "bf16", ragged=True, rot=64, pairs=True), name="append_prompt"),
        # one token over a short context
        dict(_case("attn", 1, 1, 1000, 32, 8, 128, "f32"), name="attn_token"),
        # the decode batch's attention: the cache read of a serving step
        dict(_case("attn", 64, 1, 16384, 64, 8, 128, "bf16", ragged=True), name="attn_batch"),
        # one request at a context of 128k less one: a long axis and few rows
        dict(_case("attn", 1, 1, 131071, 64, 8, 128, "bf16"), name="attn_long"),
        # speculative windows of 8 tokens, layers with a sliding window, f32 activations, 5 heads a group
        dict(_case("attn", 4, 8, 8190, 20, 4, 64, "f32", ragged=True, window=4096), name="attn_window"),
        # two prompts' chunks over their own tokens and what stood in front of them
        dict(_case("attn", 2, 4096, 6001, 32, 8, 128, "bf16", ragged=True), name="attn_prompt"),
        # selection for a decode batch at long contexts
        dict(_case("select", 16, 1, 65536, 64, 8, 128, "bf16", ragged=True, sel=32), name="select_batch"),
        # selection for every token of a prompt chunk
        dict(_case("select", 1, 4096, 16383, 32, 4, 128, "bf16", sel=16), name="select_prompt"),
        # the decode batch over its selected blocks
        dict(_case("sparse", 16, 1, 65536, 64, 8, 128, "bf16", ragged=True, sel=32), name="sparse_batch"),
        # a prompt chunk over the selected blocks of each token
        dict(_case("sparse", 1, 4096, 16383, 32, 4, 128, "bf16", sel=16), name="sparse_prompt"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        at = most.setdefault(c["op"], [0, 0, 0])
        at[0], at[1], at[2] = max(at[0], w["bytes"]), max(at[1], w["flops"]), max(at[2], c["seqs"] * c["len"] * c["kv"] * c["dim"])
    while True:
        op = rng.choice(("append", "attn", "attn", "select", "sparse"))
        kv, dim = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 128, 128, 256))
        group = rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16))
        kind = rng.choice(("token", "window", "prompt"))
        new = 1 if kind == "token" else rng.randint(2, 16) if kind == "window" else _log_int(rng, 17, 4096)
        seqs = _log_int(rng, 1, 64) if kind != "prompt" else rng.randint(1, 4)
        length = _log_int(rng, max(new, 64), 131072 if op != "append" else 16384)
        c = _case(op, seqs, new, length, kv * group, kv, dim, rng.choice(("f32", "bf16", "bf16")), ragged=rng.random() < 0.7)
        if op == "append":
            c.update(rot=rng.choice((dim, dim, dim // 2)), pairs=rng.random() < 0.5)
        if op == "attn" and rng.random() < 0.3:
            c.update(window=_log_int(rng, 64, 8192))
        if op in ("select", "sparse"):
            c.update(sel=_log_int(rng, 4, 48), first=rng.randint(0, 2), last=rng.randint(1, 2))
        w = work(c)
        if w["bytes"] > most[op][0] or w["flops"] > most[op][1] or seqs * length * kv * dim > most[op][2]:
            continue
        if op != "append" and seqs * new * length * kv * group > 2 ** 31:           # the plain form holds every score
            continue
        if 3072 in (new, length, kv * dim, kv * group * dim):
            continue
        return c


# ---------------------------------------------------------------- what a case holds
def _lengths(c):
    """(new tokens, tokens in the cache with them) of every sequence."""
    out = []
    for i in range(c["seqs"]):
        new, length = c["new"], c["len"]
        if c["ragged"] and i:
            new = max(1, round(new * (0.25 + 0.75 * (0.618034 * i % 1))))
            if i % 5 == 4 and c["new"] > 1:
                new = 0                                                             # a sequence that sits this pass out
            length = max(new, round(length * 16.0 ** -(0.754878 * i % 1)))
        out.append((new, length))
    return out


def _touched(c):
    """(sequence, block, its tokens after the pass) of every block that new tokens fall into."""
    return [(s, b, min(BLOCK, n - BLOCK * b)) for s, (new, n) in enumerate(_lengths(c)) if new
            for b in range((n - new) // BLOCK, -(-n // BLOCK))]


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = _lengths(c)
    H, KV, D, act = c["heads"], c["kv"], c["dim"], TYPES[c["act"]]
    need = [-(-n // BLOCK) for _, n in lens]
    nb, wide = sum(need) + 3, max(need)
    order = torch.randperm(nb, generator=g, device=dev, dtype=torch.int32).cpu()    # blocks in the order an allocator hands them out
    table = torch.full((c["seqs"], wide), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    N = sum(new for new, _ in lens)
    start = [0]
    for new, _ in lens:
        start.append(start[-1] + new)

    def codes(tilt):                                                                # normal values under a tight scale, each block about a mean of its own
        x = torch.empty((nb, KV, BLOCK, D), dtype=torch.uint8, device=dev)
        for a in range(0, nb, 4096):
            y = torch.randn((min(4096, nb - a), KV, BLOCK, D), generator=g, device=dev)
            if tilt:
                y += tilt * torch.randn((y.shape[0], KV, 1, D), generator=g, device=dev)
            x[a:a + 4096] = (y * 33).round_().clamp_(-127, 127).add_(128)
        return x

    def scales():
        return (0.75 + 0.5 * torch.rand((nb, KV), generator=g, device=dev)) / 33

    k, v = codes(0.5), codes(0.0)
    st = dict(case=dict(c), start=torch.tensor(start, dtype=torch.int32, device=dev), n_tokens=N,
              kv_len=torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev), max_new=max(new for new, _ in lens),
              max_len=max(n for _, n in lens), table=table.to(dev), k_scale=scales(), v_scale=scales())
    if c["op"] == "append":
        blocks = [(int(table[s, b]), n) for s, b, n in _touched(c)]
        st["blocks"] = torch.tensor([b for b, _ in blocks], dtype=torch.int32, device=dev)
        st["counts"] = torch.tensor([n for _, n in blocks], dtype=torch.int32, device=dev)
        # k_sum counts what the sequences hold before the pass
        for (new, n), row in zip(lens, table):
            full, rest = divmod(n - new, BLOCK)
            if rest:
                k[int(row[full]), :, rest:] = 128
        sums = (k.to(torch.int32) - 128).sum(2)
        for (new, n), row in zip(lens, table):
            for b in range(-(-(n - new) // BLOCK), -(-n // BLOCK)):
                sums[int(row[b])] = 0
        half = c["rot"] // 2
        angle = torch.arange(c["len"], device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        st.update(k_sum=sums.to(torch.int16), cos=angle.cos().float(), sin=angle.sin().float(),
                  q_w=1 + 0.1 * torch.randn(D, generator=g, device=dev), k_w=1 + 0.1 * torch.randn(D, generator=g, device=dev),
                  # the rows that the projections leave: queries, keys and values side by side
                  qkv=torch.randn((N, (H + 2 * KV) * D), generator=g, device=dev).to(act), q_out=torch.empty((N, H, D), dtype=act, device=dev))
    else:
        st["k_sum"] = torch.stack([(x.to(torch.int16) - 128).sum(1, dtype=torch.int16) for x in k])
        st["q"] = torch.randn((N, H, D), generator=g, device=dev).to(act)
        st["out"] = torch.empty((N, H, D), dtype=act, device=dev)
        if c["op"] in ("select", "sparse"):
            st["sel"] = torch.empty((N, KV, c["sel"]), dtype=torch.int32, device=dev)
        if c["op"] == "sparse":
            st["sel"].copy_(_plain_select(st))
    st["k"] = k.reshape(nb, KV, BLOCK, D // 64, 64).transpose(2, 3).contiguous()
    st["v"] = v.transpose(2, 3).contiguous()
    return st


# ---------------------------------------------------------------- the plain form
def _rows(st):
    """Sequence, place among its new tokens and position of every new token; and the row of every (sequence, place)."""
    c, dev = st["case"], st["start"].device
    i = torch.arange(st["n_tokens"], device=dev)
    seq = torch.searchsorted(st["start"][1:].long(), i, right=True)
    at = i - st["start"].long()[seq]
    new = (st["start"][1:] - st["start"][:-1]).long()
    return seq, at, st["kv_len"].long()[seq] - new[seq] + at


def _padded(st, x):
    """[tokens, heads, dim] -> f32 [sequence, key/value head, place * group, dim], zeros where there is no token."""
    c = st["case"]
    seq, at, _ = _rows(st)
    y = torch.zeros((c["seqs"], st["max_new"], c["heads"], c["dim"]), device=x.device)
    y[seq, at] = x.float()
    G = c["heads"] // c["kv"]
    return y.view(c["seqs"], st["max_new"], c["kv"], G, c["dim"]).permute(0, 2, 1, 3, 4).reshape(c["seqs"], c["kv"], -1, c["dim"])


def _values(st, which):
    """The cache as f32 [sequence, head, token, dim]."""
    c, t = st["case"], st["table"].clamp(min=0).long()
    x, s = st[which][t], st[which + "_scale"][t]                                     # [S, B, KV, ...]
    x = x.transpose(-3, -2).flatten(-2) if which == "k" else x.transpose(-2, -1)     # [S, B, KV, token, dim]
    x = x.float().sub_(128).mul_(s[..., None, None])
    return x.transpose(1, 2).reshape(c["seqs"], c["kv"], -1, c["dim"])


def _plain_attn(st):
    c = st["case"]
    S, KV, G, T = c["seqs"], c["kv"], c["heads"] // c["kv"], st["max_new"]
    seq, at, pos = _rows(st)
    p = torch.matmul(_padded(st, st["q"]) * c["dim"] ** -0.5, _values(st, "k").transpose(-1, -2))
    L = p.shape[-1]
    p = p.view(S, KV, T, G, L)
    limit = torch.full((S, T), -1, device=p.device, dtype=torch.long)
    limit[seq, at] = pos
    j = torch.arange(L, device=p.device)
    seen = j <= limit[..., None]
    if c["window"]:
        seen &= j > limit[..., None] - c["window"]
    seen = seen[:, None]                                                             # [S, 1, T, L]
    if c["op"] == "sparse":
        B = L // BLOCK
        pick = torch.zeros((S, T, KV, B + 1), dtype=torch.bool, device=p.device)
        pick[seq, at] = torch.zeros((st["n_tokens"], KV, B + 1), dtype=torch.bool, device=p.device).scatter_(
            2, torch.where(st["sel"] < 0, B, st["sel"]).long(), True)
        seen = seen & pick[..., :B].repeat_interleave(BLOCK, -1).transpose(1, 2)
    p.masked_fill_(~seen[:, :, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, KV, T * G, L), _values(st, "v")).view(S, KV, T, G, c["dim"])
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(S, T, c["heads"], c["dim"])[seq, at].to(TYPES[c["act"]])


def _plain_select(st):
    c = st["case"]
    S, KV, G, T, n = c["seqs"], c["kv"], c["heads"] // c["kv"], st["max_new"], c["sel"]
    seq, at, pos = _rows(st)
    q = _padded(st, st["q"])
    qs = q.abs().amax(-1, keepdim=True) * INV127
    q8 = torch.where(qs > 0, q / qs, 0.0).round_().clamp_(-127, 127)
    t = st["table"].clamp(min=0).long()
    ks = st["k_sum"][t].transpose(1, 2)                                              # [S, KV, B, dim]
    hi = torch.div(ks, 128, rounding_mode="floor")
    lo = (ks - 128 * hi).float()                                                     # whole numbers below 2^24 in each product: exact
    dots = torch.matmul(q8, hi.float().transpose(-1, -2)).int() * 128 + torch.matmul(q8, lo.transpose(-1, -2)).int()
    score = dots.float() * qs * st["k_scale"][t].transpose(1, 2)[:, :, None]
    B = score.shape[-1]
    score = score.view(S, KV, T, G, B).amax(3) + 0.0
    score = score.transpose(1, 2)[seq, at]                                           # [N, KV, B]
    b, block = torch.arange(B, device=q.device), torch.div(pos, BLOCK, rounding_mode="floor")[:, None, None]
    score = torch.where((b < c["first"]) | (b > block - c["last"]), math.inf, score)
    score = torch.where(b <= block, score, -math.inf)
    value, at = torch.sort(score, dim=-1, descending=True, stable=True)
    pick = torch.where(value > -math.inf, at, B)[..., :n]
    pick = torch.nn.functional.pad(pick, (0, n - pick.shape[-1]), value=B).sort(-1).values
    return torch.where(pick < B, pick, -1).int()


def _plain_append(st):
    c = st["case"]
    H, KV, D, rot, N = c["heads"], c["kv"], c["dim"], c["rot"], st["n_tokens"]
    seq, at, pos = _rows(st)
    x = st["qkv"].float().view(N, H + 2 * KV, D)
    q, k, v = x.split((H, KV, KV), 1)
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["pairs"] else (x[..., :rot // 2], x[..., rot // 2:rot])
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1 if c["pairs"] else -2).flatten(-2)
        return torch.cat((y, x[..., rot:]), -1)

    q, k = turned(q, st["q_w"]), turned(k, st["k_w"])
    # the touched blocks, [sequence, block among the touched]
    new = (st["start"][1:] - st["start"][:-1]).long()
    old = st["kv_len"].long() - new                                                  # tokens in front of the pass
    b0 = old // BLOCK
    wide = -(-st["max_new"] // BLOCK) + 1
    lb = b0[:, None] + torch.arange(wide, device=q.device)
    real = (new[:, None] > 0) & (lb * BLOCK < st["kv_len"].long()[:, None])
    phys = st["table"].long().gather(1, lb.clamp(max=st["table"].shape[1] - 1))
    slot = torch.arange(BLOCK, device=q.device)
    was = (lb[..., None] * BLOCK + slot < old[:, None, None])[:, :, None, :, None]   # held before the pass
    here = (lb[..., None] * BLOCK + slot < st["kv_len"].long()[:, None, None])[:, :, None, :, None]
    out = []
    for which, x in (("k", k), ("v", v)):
        codes, scale = st[which], st[which + "_scale"]
        fresh = torch.zeros((c["seqs"], wide, KV, BLOCK, D), device=q.device)
        fresh[seq, pos // BLOCK - b0[seq], :, pos % BLOCK] = x
        held = codes[phys.clamp(min=0)]
        held = held.transpose(-3, -2).flatten(-2) if which == "k" else held.transpose(-2, -1)
        held = held.float() - 128
        s0 = torch.where(was.any(3, keepdim=True), scale[phys.clamp(min=0)][..., None, None], 0.0)
        s1 = torch.maximum(s0, fresh.abs().amax((-2, -1), keepdim=True) * INV127)
        moved = torch.where(s1 > s0, torch.round(held * (s0 / s1)), held)
        put = torch.where(s1 > 0, fresh / s1, 0.0).round().clamp(-127, 127)
        now = torch.where(was, moved, torch.where(here, put, held))
        if which == "k":
            st["k_sum"][phys[real]] = torch.where(here, now, 0.0).sum(3)[real].to(torch.int16)
        raw = (now + 128).to(torch.uint8)
        raw = raw.view(*raw.shape[:4], D // 64, 64).transpose(-3, -2) if which == "k" else raw.transpose(-2, -1)
        codes[phys[real]] = raw[real]
        scale[phys[real]] = s1[real][..., 0, 0]
        n = here[real]
        out.append((torch.where(n, now[real], 0.0) * s1[real]).transpose(1, 2).bfloat16())
    mean = st["k_sum"][phys[real]].float() * st["k_scale"][phys[real]][..., None] / here[real].sum(2).float()
    return {"q": q.to(TYPES[c["act"]]), "k": out[0], "v": out[1], "mean": mean.bfloat16()}


# ---------------------------------------------------------------- one pass
def _handles(st):
    """What a program that decodes keeps: the cache, the plan of its attention layer, the rotation, this pass's batch."""
    if "attn" not in st:
        from project_maya_b200 import api
        c = st["case"]
        cache = api.KvCache(st["k"], st["v"], st["k_scale"], st["v_scale"], st["table"], k_sum=st["k_sum"])
        st["cache"] = cache
        st["attn"] = api.KvAttention(cache, c["heads"], window=c["window"], n_sel=c["sel"], n_first=c["first"], n_last=c["last"],
                                     max_tokens=st["n_tokens"])
        st["batch"] = api.AttnBatch(st["start"], st["kv_len"], st["n_tokens"], st["max_new"], st["max_len"])
        if c["op"] == "append":
            H, KV, D = c["heads"], c["kv"], c["dim"]
            st["rope"] = api.Rope(st["cos"], st["sin"], q_w=st["q_w"], k_w=st["k_w"], eps=EPS, pairs=c["pairs"])
            st["q_in"], st["k_in"], st["v_in"] = st["qkv"].view(-1, H + 2 * KV, D).split((H, KV, KV), 1)
            n = len(st["blocks"])
            st["read"] = [torch.empty((n, BLOCK, KV, D), dtype=torch.bfloat16, device=st["k"].device) for _ in range(2)]
            st["read"].append(torch.empty((n, KV, D), dtype=torch.bfloat16, device=st["k"].device))
    return st["attn"], st["batch"]


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "append":
            return _plain_append(state)
        return _plain_select(state) if op == "select" else _plain_attn(state)
    attn, batch = _handles(state)
    if op == "append":
        q = attn.append(batch, state["q_in"], state["k_in"], state["v_in"], state["rope"], q_out=state["q_out"])
        k, v, mean = state["cache"].read(state["blocks"], state["counts"], *state["read"])
        return {"q": q, "k": k, "v": v, "mean": mean}
    if op == "select":
        return attn.select(batch, state["q"], sel=state["sel"])
    return attn.forward(batch, state["q"], sel=state["sel"] if op == "sparse" else None, out=state["out"])


def work(case):
    c = case
    H, KV, D, es = c["heads"], c["kv"], c["dim"], 4 if c["act"] == "f32" else 2
    lens = _lengths(c)
    N = sum(new for new, _ in lens)
    if c["op"] == "append":
        n = sum(k for _, _, k in _touched(c))                                        # tokens read back
        t = len(_touched(c))
        return {"bytes": N * ((2 * H + 2 * KV) * D * es + 2 * KV * D + 4 * c["rot"]) + n * KV * D * (2 + 2 * 2) + t * KV * (D * 4 + 8),
                "flops": N * (H + KV) * D * 8 + N * KV * D * 2}
    seen = read = picked = 0
    for new, n in lens:
        first = n - new
        if new == 0:
            continue
        if c["op"] == "attn":
            w = c["window"]
            for at in (range(first, n) if w else ()):
                seen += min(at + 1, w)
            seen += 0 if w else new * (first + 1 + n) // 2
            read += min(n, new - 1 + w) if w else n
        else:
            for at in range(first, n):
                b = at // BLOCK
                seen += min(at + 1, (min(c["sel"], b + 1) - 1) * BLOCK + at % BLOCK + 1)
                picked += max(0, b + 1 - c["first"] - c["last"])
            read += min(n, new * c["sel"] * BLOCK)
    if c["op"] == "select":
        blocks = sum(-(-n // BLOCK) for new, n in lens if new)
        return {"bytes": N * H * D * es + blocks * KV * (2 * D + 4) + N * KV * c["sel"] * 4, "flops": picked * H * D * 2}
    more = N * KV * c["sel"] * 4 if c["op"] == "sparse" else 0
    return {"bytes": 2 * N * H * D * es + read * KV * (2 * D + 8 / BLOCK) + more, "flops": 4 * seen * H * D}


# ---------------------------------------------------------------- from the definition, in 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "select":                                                          # whole numbers: nothing is rounded
        return None
    st = prepare(c, seed)
    H, KV, D, G = c["heads"], c["kv"], c["dim"], c["heads"] // c["kv"]
    lens, table = _lengths(c), st["table"].tolist()
    if c["op"] != "append":
        out = torch.zeros((st["n_tokens"], H, D), dtype=torch.float64, device="cuda")
        row = 0
        for s, (new, n) in enumerate(lens):
            if not new:
                continue
            ids = torch.tensor(table[s][:-(-n // BLOCK)], device="cuda")
            j = torch.arange(n, device="cuda")
            for h in range(KV):
                k = torch.cat([st["k"][ids, h, x].reshape(-1, 64) for x in range(D // 64)], 1)[:n].double() - 128
                v = st["v"][ids, h].permute(0, 2, 1).reshape(-1, D)[:n].double() - 128
                k *= st["k_scale"][ids, h].double().repeat_interleave(BLOCK)[:n, None]
                v *= st["v_scale"][ids, h].double().repeat_interleave(BLOCK)[:n, None]
                for a in range(0, new, 512):
                    e = min(new, a + 512)
                    at = torch.arange(n - new + a, n - new + e, device="cuda")[:, None]
                    ok = j <= at
                    if c["window"]:
                        ok &= at - j < c["window"]
                    if c["op"] == "sparse":
                        sel = st["sel"][row + a:row + e, h].long()
                        has = torch.zeros((e - a, len(ids) + 1), dtype=torch.bool, device="cuda")
                        has[torch.arange(e - a, device="cuda")[:, None], torch.where(sel < 0, len(ids), sel)] = True
                        ok = ok & has[:, j // BLOCK]
                    q = st["q"][row + a:row + e, h * G:(h + 1) * G].double()
                    logits = torch.einsum("tgd,nd->tgn", q, k) / math.sqrt(D)
                    weight = torch.softmax(logits.masked_fill(~ok[:, None], -math.inf), -1)
                    out[row + a:row + e, h * G:(h + 1) * G] = torch.einsum("tgn,nd->tgd", weight, v)
            row += new
        return out
    x = st["qkv"].double().view(-1, H + 2 * KV, D)
    at = torch.cat([torch.arange(n - new, n) for new, n in lens]).cuda()
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
    half = c["rot"] // 2

    def head(y, w):
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        z = y[..., :c["rot"]]
        z = torch.view_as_complex(z.reshape(*z.shape[:-1], half, 2).contiguous()) if c["pairs"] else torch.complex(z[..., :half], z[..., half:])
        z = torch.view_as_real(z * turn)
        y[..., :c["rot"]] = z.flatten(-2) if c["pairs"] else torch.cat((z[..., 0], z[..., 1]), -1)
        return y

    q, k, v = head(x[:, :H].clone(), st["q_w"]), head(x[:, H:H + KV].clone(), st["k_w"]), x[:, H + KV:]
    ks, vs, means = [], [], []
    row = {}
    for s, (new, _) in enumerate(lens):
        row[s] = sum(m for m, _ in lens[:s])
    for s, b, n in _touched(c):
        new, length = lens[s]
        id_, first = table[s][b], length - new
        held = max(0, min(n, first - b * BLOCK))                                     # tokens of the block from before
        a = row[s] + max(0, b * BLOCK - first)
        for name, src, into in (("k", k, ks), ("v", v, vs)):
            fresh = src[a:a + n - held]                                              # [tokens, KV, D]
            codes = st[name][id_].double() - 128
            codes = codes.permute(2, 0, 1, 3).reshape(BLOCK, KV, D) if name == "k" else codes.permute(2, 0, 1)
            s0 = st[name + "_scale"][id_].double()[:, None] if held else torch.zeros((KV, 1), dtype=torch.float64, device="cuda")
            s1 = torch.maximum(s0, fresh.abs().amax((0, 2))[:, None] / 127)
            whole = torch.zeros((BLOCK, KV, D), dtype=torch.float64, device="cuda")
            whole[:held] = torch.round(codes[:held] * (s0 / s1))
            whole[held:n] = torch.round(fresh / s1)
            into.append(whole * s1)
        means.append(ks[-1].sum(0) / n)
    return {"q": q, "k": torch.stack(ks), "v": torch.stack(vs), "mean": torch.stack(means)}
