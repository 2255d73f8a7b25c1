"""A whole decoder layer over resident GGUF weights: attention over the 8-bit cache, then the routed experts.

    python -m project_maya_b200.decoder_layer [--tokens N] [--steps N] [--long]

runs one layer of random weights over a prompt and then token by token, and prints what each half takes.

    h -> RMS norm -> q8_1 -> [q | k | v] rows (GGUF product) -> norms of the heads, rotation, cache append
      -> attention (over the blocks that select() chooses, for single tokens of contexts of `sparse_from` tokens and more) -> output rows (GGUF product)
    h + attention -> RMS norm, router logits -> experts -> h
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass

import torch

from . import api


@dataclass
class AttentionConfig:
    n_embd: int
    n_q: int
    n_kv: int
    head_dim: int
    weight_type: int = api.Q8_0          # of the projections
    rot_dim: int = 0                     # 0: all of head_dim
    theta: float = 10000.0
    eps: float = 1e-6
    n_sel: int = 0                       # blocks a token reads in a long context; 0: all of them always
    sparse_from: int = 8192              # tokens of its own context from which on a sequence's single token reads selected blocks
    rows: torch.dtype = torch.float32    # of queries, keys, values and outputs between the products: f32 (P in 22 bits), or bf16 (P in 11; prompts on tcgen05)

    def __post_init__(self):
        assert self.rows in (torch.float32, torch.bfloat16)

    @property
    def qkv_rows(self) -> int:
        return (self.n_q + 2 * self.n_kv) * self.head_dim


class DecoderLayer:
    """w_qkv uint8: qkv_rows GGUF rows of n_embd values, [q | k | v]; w_o: n_embd rows of n_q * head_dim values; norms f32 (in, post: [n_embd];
    q, k: [head_dim]); router_w [n_expert, n_embd] f32; experts as for api.MoeLayer.  `table` i32 [n_seq, blocks of a sequence] hands out the
    cache's blocks; max_tokens: the longest context; max_chunk: the longest prompt chunk."""

    def __init__(self, cfg: AttentionConfig, moe_cfg: api.MoeLayerConfig, w_qkv, w_o, norms: dict, router_w, experts, table, n_blocks: int,
                 max_tokens: int, max_chunk: int = 1024):
        c, dev = cfg, w_qkv.device
        self.cfg, self.moe_cfg, self.w_qkv, self.w_o, self.norms, self.router_w = cfg, moe_cfg, w_qkv, w_o, norms, router_w
        half = (c.rot_dim or c.head_dim) // 2
        positions = max(max_tokens, table.shape[1] * api.KV_BLOCK)             # all that the table's blocks hold
        angle = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * c.theta ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        self.rope = api.Rope(angle.cos().float(), angle.sin().float(), q_w=norms["q"], k_w=norms["k"], eps=c.eps)
        self.cache = api.KvCache.empty(n_blocks, c.n_kv, c.head_dim, table, sums=c.n_sel > 0)
        self.attn = api.KvAttention(self.cache, c.n_q, n_sel=c.n_sel)
        self.token = api.MoeLayer(moe_cfg, experts)
        self.chunk = api.MoePrefill(moe_cfg, experts, max_tokens=max_chunk)
        self.bounds = {}

    def _product(self, w, x, n_out: int):
        """x [T, n_in] f32 times GGUF rows: the decode GEMV for up to 8 tokens, the prompt path's GEMM beyond."""
        (T, n_in), t = x.shape, self.cfg.weight_type
        if T <= api.MAX_COLS:
            return api.native_mmvq(t, w, api.native_quantize_q8_1(x), n_in, n_out, T)
        if T not in self.bounds:
            self.bounds[T] = torch.tensor([0, T], dtype=torch.int32, device=x.device)
        y = torch.empty((T, n_out), dtype=torch.float32, device=x.device)
        api.mmq_run(api.mmq_product(w, t, n_out, n_in, w.numel(), 1, api.mmq_quantize(x, None, t), self.bounds[T], None, T, y, n_out))
        return y

    def _rms(self, h, w):
        return h * torch.rsqrt((h * h).mean(-1, keepdim=True) + self.cfg.eps) * w

    def attention(self, h, batch: api.AttnBatch):
        """The attention half for the batch's new tokens: h [T, n_embd] f32 -> what is added to it.  The cache holds their keys and values
        afterwards."""
        c, T = self.cfg, h.shape[0]
        rows = self._product(self.w_qkv, self._rms(h, self.norms["in"]), c.qkv_rows).view(T, -1, c.head_dim)
        q, k, v = rows.to(c.rows).split((c.n_q, c.n_kv, c.n_kv), 1)
        out = self._attend(batch, self.attn.append(batch, q, k, v, self.rope))
        return self._product(self.w_o, out.view(T, -1).float(), c.n_embd)

    def _attend(self, batch: api.AttnBatch, q):
        """Attention over every block, or over selected ones for the single tokens of contexts of `sparse_from` tokens and more."""
        c, b = self.cfg, batch.desc
        if c.n_sel == 0 or b.max_new > 1 or b.max_len < c.sparse_from:
            return self.attn.forward(batch, q)
        if batch.min_len >= c.sparse_from:
            return self.attn.forward(batch, q, sel=self.attn.select(batch, q))
        # Lengths on both sides, or not known here: a pass for each side in which the other's sequences have no tokens, whose rows are zeros then.
        long = batch.kv_len >= c.sparse_from
        far = api.AttnBatch(batch.start, torch.where(long, batch.kv_len, 0), b.n_tokens, 1, b.max_len)
        near = api.AttnBatch(batch.start, torch.where(long, 0, batch.kv_len), b.n_tokens, 1, c.sparse_from - 1)
        return self.attn.forward(far, q, sel=self.attn.select(far, q)) + self.attn.forward(near, q)

    def forward(self, h, batch: api.AttnBatch):
        a = self.attention(h, batch)
        if h.shape[0] == 1:
            h_out = torch.empty_like(h)
            x, logits = api.rms_router(h[0], a[0], self.norms["post"], self.cfg.eps, self.router_w, h_out=h_out[0])
            return h_out + self.token.forward(logits[None], x[None])[2]
        h = h + a
        x = self._rms(h, self.norms["post"])
        logits = torch.mm(x, self.router_w.t())
        if h.shape[0] <= self.token.max_tokens:
            return h + self.token.forward(logits, x)[2]
        return h + self.chunk.forward(logits, x)[2]


def synthetic_layer(cfg: AttentionConfig, moe_cfg: api.MoeLayerConfig, max_tokens: int, max_chunk: int, n_seq: int = 1, seed: int = 1) -> DecoderLayer:
    """A layer of N(0, 0.02) weights quantized by the library, its cache's blocks handed out in random order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w_qkv = api.synth_weights(cfg.weight_type, seed, 0.02, cfg.qkv_rows, cfg.n_embd)
    w_o = api.synth_weights(cfg.weight_type, seed + 1, 0.02, cfg.n_embd, cfg.n_q * cfg.head_dim)
    experts = torch.empty((moe_cfg.n_expert, moe_cfg.blob_bytes), dtype=torch.uint8, device="cuda")
    gu = 2 * moe_cfg.n_ff * api.row_bytes(moe_cfg.gu_type, moe_cfg.n_embd)
    for e in range(moe_cfg.n_expert):
        api.synth_weights(moe_cfg.gu_type, seed + 2 * e + 10, 0.02, 2 * moe_cfg.n_ff, moe_cfg.n_embd, experts[e, :gu])
        api.synth_weights(moe_cfg.d_type, seed + 2 * e + 11, 0.02, moe_cfg.n_embd, moe_cfg.n_ff, experts[e, gu:])
    norms = {name: 1 + 0.1 * torch.randn(n, generator=g, device="cuda")
             for name, n in (("in", cfg.n_embd), ("post", cfg.n_embd), ("q", cfg.head_dim), ("k", cfg.head_dim))}
    router_w = torch.randn((moe_cfg.n_expert, cfg.n_embd), generator=g, device="cuda") / cfg.n_embd ** 0.5
    wide = -(-max_tokens // api.KV_BLOCK)
    table = torch.randperm(n_seq * wide, generator=g, device="cuda", dtype=torch.int32).view(n_seq, wide).contiguous()
    return DecoderLayer(cfg, moe_cfg, w_qkv, w_o, norms, router_w, experts, table, n_seq * wide, max_tokens, max_chunk)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=4096, help="prompt tokens")
    ap.add_argument("--steps", type=int, default=64, help="tokens decoded after it")
    ap.add_argument("--long", action="store_true", help="tokens read 32 selected blocks from 2048 tokens of context on")
    a = ap.parse_args()
    cfg = AttentionConfig(4096, 32, 8, 128, n_sel=32 if a.long else 0, sparse_from=2048, rows=torch.bfloat16)
    moe = api.MoeLayerConfig(4096, 1536, 64, 8, api.Q4_K, api.Q4_K)
    layer = synthetic_layer(cfg, moe, a.tokens + a.steps, max(a.tokens, 32))
    h = torch.randn((a.tokens + a.steps, cfg.n_embd), device="cuda")

    def timed(fn, n):
        fn()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(n):
            fn()
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end) / n * 1e3

    prompt = api.AttnBatch.of([a.tokens], [a.tokens])
    both, half = timed(lambda: layer.forward(h[:a.tokens], prompt), 5), timed(lambda: layer.attention(h[:a.tokens], prompt), 5)
    print(f"prompt of {a.tokens} tokens: {both:.1f} us a layer, of it attention {half:.1f} us")
    steps = [api.AttnBatch.of([1], [a.tokens + i + 1]) for i in range(a.steps)]
    run = lambda fn: [fn(h[a.tokens + i:a.tokens + i + 1], b) for i, b in enumerate(steps)]   # noqa: E731
    both, half = timed(lambda: run(layer.forward), 3) / a.steps, timed(lambda: run(layer.attention), 3) / a.steps
    print(f"token behind it: {both:.1f} us a layer, of it attention {half:.1f} us")
    assert layer.attn.error() == 0 and layer.chunk.error() == 0 and layer.token.error() == 0


if __name__ == "__main__":
    main()
