"""Host-side mirror of the reference's per-layer expert-FFN entry points, over the C ABI (include/maya_moe.h).

Names, argument meaning and error behaviour follow the reference's C++ free functions (namespace strata::kernels,
strata::kernels::glmf): device buffers in, device buffers out, an explicit stream, nothing allocated by the callee.
torch is used only for device memory and streams: every function takes torch CUDA tensors (or raw integer device
addresses) and launches this library's own CUDA kernels.  A negative status raises MayaError, as the reference's
`native_*` family throws std::invalid_argument / std::runtime_error (native_mmvq.cu:1080-1099).
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import AttnArgs, AttnBatchDesc, ExpertLayout, HcPostArgs, KvCacheDesc, KvPagesDesc, LoraArgs, MmqProduct, MoeLayerDesc, MoePlan, MoeWin, RmsArgs, RopeArgs, RouteArgs, SelectArgs

Q8_0, Q4_K, IQ3_S, IQ2_S = 8, 12, 21, 22
Q5_K, Q6_K, IQ2_XXS, IQ3_XXS, IQ1_S, IQ4_XS = 13, 14, 16, 18, 19, 23      # decode paths only (see maya_ggml_type in the header)
_BLOCK = {Q8_0: 32, Q4_K: 256, IQ3_S: 256, IQ2_S: 256, Q5_K: 256, Q6_K: 256, IQ2_XXS: 256, IQ3_XXS: 256, IQ4_XS: 256, IQ1_S: 256}   # values per GGUF block
TYPE_NAMES = {Q8_0: "Q8_0", Q4_K: "Q4_K", IQ3_S: "IQ3_S", IQ2_S: "IQ2_S", Q5_K: "Q5_K", Q6_K: "Q6_K", IQ2_XXS: "IQ2_XXS",
              IQ3_XXS: "IQ3_XXS", IQ4_XS: "IQ4_XS", IQ1_S: "IQ1_S"}
STATUS = {0: "ok", -1: "bad argument", -2: "unsupported ggml type", -3: "CUDA launch failed", -4: "beyond a limit",
          -5: "no sm_100 device"}
LAYER_CHOICE, LAYER_FUSED, LAYER_TOKEN, LAYER_STAGED = 0, 1, 2, 3        # maya_layer_kernel
XQ_Q8_1, XQ_MMQ = 1, 2        # 8-bit rows: q8_1 blocks (native_mmvq reads them), the prompt path's image (mmq_run) - enum maya_xq_image
INF = float("inf")
MAX_COLS = 8                 # activation columns of native_mmvq (MAYA_MAX_COLS)


class MayaError(RuntimeError):
    def __init__(self, what: str, status: int):
        super().__init__(f"{what}: {STATUS.get(status, status)} (status {status})")
        self.status = status


def _check(what: str, status: int) -> None:
    if status != 0:
        raise MayaError(what, status)


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    assert t.is_cuda and t.is_contiguous(), "device-contiguous tensor expected"
    return t.data_ptr()


def _stream(stream=None) -> int:
    if stream is None:           # the current stream's handle, without the Stream object (0.2 us instead of 3.1: a small layer's token takes 18)
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _here(what: str, *tensors, stream=None) -> int:
    """Tensors of a call: all on the current device, on whose current stream (or `stream`) it goes; returns that stream's handle."""
    dev = torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -2
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise MayaError(f"{what}: tensors of the current device expected", -1)
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else _stream(stream)


# ---------------------------------------------------------------- formats (host only: usable without a GPU)
def row_bytes(ggml_type: int, n: int) -> int:
    return int(_lib.load().maya_row_bytes(ggml_type, n))


def q8_1_bytes(n_in: int, ncols: int = 1) -> int:
    return int(_lib.load().maya_q8_1_bytes(n_in, ncols))


def native_expert_layout(gu_type: int, d_type: int, n_embd: int, n_ff: int, up_type: int | None = None) -> ExpertLayout:
    L = ExpertLayout()
    _check("native_expert_layout", _lib.load().maya_expert_layout_make(gu_type, gu_type if up_type is None else up_type,
                                                                       d_type, n_embd, n_ff, C.byref(L)))
    return L


def quantize_weights_host(ggml_type: int, w) -> "torch.Tensor":
    """Host f32 rows [n_rows, n_cols] -> uint8 [n_rows, row_bytes] of GGUF blocks (this library's own quantizers)."""
    w = torch.as_tensor(w, dtype=torch.float32).contiguous().cpu()
    n_rows, n_cols = w.shape
    out = torch.empty((n_rows, row_bytes(ggml_type, n_cols)), dtype=torch.uint8)
    _check("quantize_weights_host",
           _lib.load().maya_quantize_weights_host(ggml_type, w.data_ptr(), n_rows, n_cols, out.data_ptr()))
    return out


def synth_weights(ggml_type: int, seed: int, sigma: float, n_rows: int, n_cols: int, out=None, stream=None):
    """Device: n_rows x n_cols N(0, sigma) weights quantized to ggml_type, written as blocks into `out` (uint8)."""
    nbytes = n_rows * row_bytes(ggml_type, n_cols)
    if out is None:
        out = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    _check("synth_weights", _lib.load().maya_synth_weights(ggml_type, seed, sigma, n_rows, n_cols, _ptr(out), _stream(stream)))
    return out


# ---------------------------------------------------------------- router
def router_top10(logits, k: int, ids=None, weights=None, stream=None):
    """router_top10 (router_top10.hpp:17).  logits [n_tokens, n_expert] f32 -> ids i32, weights f32 [n_tokens, k]."""
    T, E = logits.shape
    ids = ids if ids is not None else torch.empty((T, k), dtype=torch.int32, device=logits.device)
    weights = weights if weights is not None else torch.empty((T, k), dtype=torch.float32, device=logits.device)
    _check("router_top10", _lib.load().maya_router_top10(_ptr(logits), T, E, k, _ptr(ids), _ptr(weights), _stream(stream)))
    return ids, weights


def router_sigmoid(logits, bias, k: int, w_scale: float = 1.0, norm_w: bool = True, stream=None):
    T, E = logits.shape
    ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
    weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    _check("router_sigmoid", _lib.load().maya_router_sigmoid(_ptr(logits), _ptr(bias), T, E, k, w_scale, int(norm_w),
                                                             _ptr(ids), _ptr(weights), _stream(stream)))
    return ids, weights


@dataclass
class GroupRouting:
    """How router_groups chooses: n_group groups of neighbouring experts of which the n_keep best are kept (1, 1: no groups), bias f32 [n_expert] or
    None, sigmoid or softmax scores, top2: a group scores the sum of its two highest (else its highest), norm_w and w_scale of the weights."""
    n_group: int = 1
    n_keep: int = 1
    bias: "torch.Tensor | None" = None
    sigmoid: bool = True
    top2: bool = True
    norm_w: bool = True
    w_scale: float = 1.0

    def route(self, logits, k: int, ids=None, weights=None, stream=None):
        return router_groups(logits, k, self.n_group, self.n_keep, self.bias, self.sigmoid, self.top2, self.norm_w, self.w_scale, ids, weights, stream)


def router_groups(logits, k: int, n_group: int = 1, n_keep: int = 1, bias=None, sigmoid: bool = True, top2: bool = True, norm_w: bool = True,
                  w_scale: float = 1.0, ids=None, weights=None, stream=None):
    """No counterpart in the reference.  logits [T, n_expert] f32 -> ids i32, weights f32 [T, k]: scores s = sigmoid or softmax of the logits, choice by
    s + bias - the n_keep best of n_group groups, then the k best of their experts - and weights s / max(their sum, 2^-14) * w_scale (norm_w False:
    s * w_scale).  include/maya_moe.h states it in full (maya_router_groups)."""
    T, E = logits.shape
    s = _here("router_groups", logits, bias, ids, weights, stream=stream)
    assert logits.dtype is torch.float32 and (bias is None or (bias.dtype is torch.float32 and bias.numel() == E))
    if weights is None:
        weights = logits.new_empty((T, k))
    if ids is None:
        ids = torch.empty_like(weights, dtype=torch.int32)
    assert ids.dtype is torch.int32 and weights.dtype is torch.float32 and ids.numel() == weights.numel() == T * k
    a = RouteArgs(_ptr(logits), _ptr(bias), T, E, k, n_group, n_keep, sigmoid, top2, norm_w, w_scale, _ptr(ids), _ptr(weights))
    _check("router_groups", _lib.load().maya_router_groups(C.byref(a), s))
    return ids, weights


# ---------------------------------------------------------------- activations
def native_quantize_q8_1(x, out=None, stream=None):
    """native_quantize_q8_1 (native_mmvq.hpp:38).  x [ncols, n_in] f32 or bf16 -> uint8 [ncols, n_in/32*36]."""
    x2 = x.reshape(-1, x.shape[-1])
    ncols, n_in = x2.shape
    out = out if out is not None else torch.empty((ncols, n_in // 32 * 36), dtype=torch.uint8, device=x.device)
    lib = _lib.load()
    if x.dtype == torch.bfloat16:
        _check("quantize_q8_1", lib.maya_quantize_q8_1_bf16(_ptr(x2), _ptr(out), n_in, ncols, _stream(stream)))
    else:
        assert x.dtype == torch.float32
        _check("quantize_q8_1", lib.maya_quantize_q8_1(_ptr(x2), _ptr(out), n_in, ncols, _stream(stream)))
    return out


def swiglu_q8_1(gate, up, limit: float = INF, out=None, stream=None):
    n = gate.numel()
    out = out if out is not None else torch.empty(n // 32 * 36, dtype=torch.uint8, device=gate.device)
    _check("swiglu_q8_1", _lib.load().maya_swiglu_q8_1(_ptr(gate), _ptr(up), limit, n, _ptr(out), _stream(stream)))
    return out


# ---------------------------------------------------------------- GEMV
def native_mmvq(ggml_type: int, weights, x_q8_1, n_in: int, n_out: int, ncols: int = 1, y=None, stream=None):
    """native_mmvq (native_mmvq.hpp:109) / iq_mmvq (iq_kernels.hpp:24): y [ncols, n_out] f32."""
    y = y if y is not None else torch.empty((ncols, n_out), dtype=torch.float32, device="cuda")
    _check("native_mmvq", _lib.load().maya_mmvq(ggml_type, _ptr(weights), _ptr(x_q8_1), _ptr(y), n_in, n_out, ncols,
                                               _stream(stream)))
    return y


# ---------------------------------------------------------------- low-rank adapters
LORA_CHOICE, LORA_FEW, LORA_MANY = 0, 1, 2               # maya_lora_kernel


class LoraAdapters:
    """Low-rank adapters of one projection, of which every token uses its own or none: out[t] = y[t] + scale[i] * b[i] (a[i] x[t]), i = idx[t].

    a [n, rank, n_in] and b [n, n_out, rank] bf16 or f16, scale f32 [n] or None (1); they are kept as they are, or - where the rank is not a multiple
    of 16 - as copies padded with zeros (an infinite x makes NaN with them).  n_in % 32 == 0, rank <= 256.  max_tokens sizes the scratch, which belongs to this object: one thread and one
    stream at a time."""

    def __init__(self, a, b, scale=None, max_tokens: int = 4096):
        n, rank, n_in = a.shape
        n_out = b.shape[1]
        assert b.shape == (n, n_out, rank) and a.dtype is b.dtype and a.dtype in (torch.bfloat16, torch.float16)
        assert scale is None or (scale.dtype is torch.float32 and scale.shape == (n,))
        assert b.device == a.device and (scale is None or scale.device == a.device), "a, b and scale of one device expected"
        wide = -(-rank // 16) * 16
        if wide != rank:
            a, b = torch.nn.functional.pad(a, (0, 0, 0, wide - rank)), torch.nn.functional.pad(b, (0, wide - rank))
        self.a, self.b, self.scale, self.rank, self.n_in, self.n_out, self.max_tokens = a, b, scale, wide, n_in, n_out, max_tokens
        nbytes = int(_lib.load().maya_lora_scratch_bytes(n_in, wide, n, max_tokens))
        if nbytes == 0:
            raise MayaError("lora_scratch_bytes", -1)
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=a.device)
        self.scratch[:256].zero_()
        self._fixed = _ptr(a), _ptr(b), _ptr(scale)
        self._sizes = n_in, n_out, wide, n

    def forward(self, x, idx, y=None, out=None, kernel: int = LORA_CHOICE, stream=None):
        """x [T, n_in] f32 or bf16, idx i32 [T] (outside 0 .. n - 1: no adapter), y f32 [T, n_out] (None: zeros) -> out f32 [T, n_out], which may be y.
        kernel: LORA_FEW (each token by itself), LORA_MANY (tiles of one adapter's tokens) or the sizes' choice."""
        s = _here("lora", self.scratch, x, idx, y, out, stream=stream)
        T = x.shape[0]
        if out is None:
            out = torch.empty((T, self.n_out), dtype=torch.float32, device=x.device)
        assert idx.dtype is torch.int32 and idx.shape == (T,) and out.dtype is torch.float32 and (y is None or y.dtype is torch.float32)
        xp, ld_x = _matrix(x, (T, self.n_in))
        op, ld_out = _matrix(out, (T, self.n_out))
        yp, ld_y = (None, self.n_out) if y is None else _matrix(y, (T, self.n_out))
        a, b, scale = self._fixed
        args = LoraArgs(xp, yp, op, a, b, scale, _ptr(idx), self.scratch.data_ptr(), self.scratch.numel(), ld_x, ld_y, ld_out, T, *self._sizes,
                        x.dtype is torch.bfloat16, self.a.dtype is torch.float16, kernel)
        _check("lora", _lib.load().maya_lora(C.byref(args), s))
        return out

    def error(self, stream=None) -> int:
        """1 after a call whose bounded wait ran out (its output is not valid); synchronises the stream.  The word is zeroed then."""
        code = int(_lib.load().maya_lora_error(self.scratch.data_ptr(), _stream(stream)))
        if code < 0:
            raise MayaError("lora_error", code)
        if code > 0:
            self.scratch[:4].zero_()
            torch.cuda.current_stream(self.scratch.device).synchronize()
        return code


# ---------------------------------------------------------------- decode experts
def make_plan(plan_ptr, plan_w, cpu_part=None, cpu_flag=None, skip=None) -> MoePlan:
    return MoePlan(_ptr(plan_ptr), _ptr(plan_w), _ptr(cpu_part), _ptr(cpu_flag), _ptr(skip))


def moe_gate_up(gu_type: int, plan: MoePlan, k: int, n_embd: int, n_ff: int, limit: float, xq, hq, sh_down=None,
                sh_type: int = 0, sh_hq=None, n_ff_sh: int = 0, sh_out=None, stream=None) -> None:
    """glmf::moe_gate_up (glm_fast.hpp:496)."""
    _check("moe_gate_up", _lib.load().maya_moe_gate_up(gu_type, C.byref(plan), k, n_embd, n_ff, limit, _ptr(xq), _ptr(hq),
                                                      _ptr(sh_down), sh_type, _ptr(sh_hq), n_ff_sh, _ptr(sh_out),
                                                      _stream(stream)))


def moe_down(d_type: int, plan: MoePlan, k: int, n_embd: int, n_ff: int, down_off: int, hq, sh_out, out, stream=None) -> None:
    """glmf::moe_down (glm_fast.hpp:499)."""
    _check("moe_down", _lib.load().maya_moe_down(d_type, C.byref(plan), k, n_embd, n_ff, down_off, _ptr(hq), _ptr(sh_out),
                                                _ptr(out), _stream(stream)))


def moe_win_experts(gu_type: int, d_type: int, win: MoeWin, stream=None) -> None:
    """glmf::moe_win_experts (glm_fast.hpp:465)."""
    _check("moe_win_experts", _lib.load().maya_moe_win_experts(gu_type, d_type, C.byref(win), _stream(stream)))


def moe_win_experts_checked(gu_type: int, d_type: int, win: MoeWin, polls: int, error=None, stream=None) -> None:
    """moe_win_experts with the caller's bound on the waits for weight rows; error: int32 [1], set to 1 when one ran out."""
    _check("moe_win_experts_checked",
           _lib.load().maya_moe_win_experts_checked(gu_type, d_type, C.byref(win), polls, _ptr(error), _stream(stream)))


def native_expert_scratch_bytes(cap_entries: int, n_ff: int) -> int:
    return int(_lib.load().maya_expert_scratch_bytes(cap_entries, n_ff))


def native_expert_grouped(L: ExpertLayout, grp_ptr, grp_start, n_groups, ent_dst, ent_tok, cap_groups: int,
                          cap_entries: int, x_q8_1, scratch, out, swiglu_limit: float = INF, stream=None) -> None:
    """native_expert_grouped (iq_kernels.hpp:89)."""
    _check("native_expert_grouped",
           _lib.load().maya_expert_grouped(C.byref(L), _ptr(grp_ptr), _ptr(grp_start), _ptr(n_groups), _ptr(ent_dst),
                                           _ptr(ent_tok), cap_groups, cap_entries, _ptr(x_q8_1), _ptr(scratch), _ptr(out),
                                           _stream(stream), swiglu_limit))


def native_expert_grouped_static(L: ExpertLayout, grp_ptr, grp_start, n_groups, ent_dst, ent_tok, cap_groups: int,
                                 cap_entries: int, x_q8_1, out, swiglu_limit: float = INF, stream=None) -> None:
    """native_expert_grouped without a scratch argument: for callers that cannot allocate or pass device scratch.
    The q8_1 image of h lives in a 2 MiB array built into the library (see maya_expert_grouped_static in the header:
    size limit, first call outside stream capture, calls on one GPU must not overlap)."""
    _check("native_expert_grouped_static",
           _lib.load().maya_expert_grouped_static(C.byref(L), _ptr(grp_ptr), _ptr(grp_start), _ptr(n_groups), _ptr(ent_dst),
                                                  _ptr(ent_tok), cap_groups, cap_entries, _ptr(x_q8_1), _ptr(out),
                                                  _stream(stream), swiglu_limit))


def moe_combine(parts, weights, shared, n_embd: int, k: int, n_tok: int = 1, y=None, stream=None):
    """native_moe_combine[_multi] (native_moe.hpp:16-20) / moe_combine (shared_expert.hpp:98)."""
    y = y if y is not None else torch.empty((n_tok, n_embd), dtype=torch.float32, device="cuda")
    _check("moe_combine", _lib.load().maya_moe_combine(_ptr(parts), _ptr(weights), _ptr(shared), _ptr(y), n_embd, k, n_tok,
                                                      _stream(stream)))
    return y


# ---------------------------------------------------------------- prefill grouping
def expert_group(ids, n_expert: int, stream=None):
    """glmb::expert_count + the device-side bounds scan + glmb::expert_scatter.  ids [T, k] i32 ->
    (counts [E], bounds [E + 1], pos [T * k], row_tok [T * k]) with no host round trip."""
    T, k = ids.shape
    n = T * k
    dev = ids.device
    counts = torch.empty(n_expert, dtype=torch.int32, device=dev)
    rank = torch.empty(n, dtype=torch.int32, device=dev)
    bounds = torch.empty(n_expert + 1, dtype=torch.int32, device=dev)
    pos = torch.empty(n, dtype=torch.int32, device=dev)
    row_tok = torch.empty(n, dtype=torch.int32, device=dev)
    lib, s = _lib.load(), _stream(stream)
    _check("expert_count", lib.maya_expert_count(_ptr(ids), n, n_expert, _ptr(counts), _ptr(rank), s))
    _check("expert_bounds", lib.maya_expert_bounds(_ptr(counts), n_expert, _ptr(bounds), s))
    _check("expert_scatter", lib.maya_expert_scatter(_ptr(ids), _ptr(rank), _ptr(bounds), n, k, _ptr(row_tok), _ptr(pos), s))
    return counts, bounds, pos, row_tok


def swiglu_rows(gu, n_ff: int, limit: float = INF, stream=None):
    rows = gu.shape[0]
    h = torch.empty((rows, n_ff), dtype=torch.float32, device=gu.device)
    _check("swiglu_rows", _lib.load().maya_swiglu_rows(_ptr(gu), _ptr(h), rows, n_ff, limit, 0, _stream(stream)))
    return h


def moe_combine_rows(out, pos, w, sh, T: int, k: int, n_embd: int, stream=None):
    ffn = torch.empty((T, n_embd), dtype=torch.float32, device=out.device)
    _check("moe_combine_rows", _lib.load().maya_moe_combine_rows(_ptr(out), _ptr(pos), _ptr(w), _ptr(sh), T, k, n_embd,
                                                                _ptr(ffn), _stream(stream)))
    return ffn


# ---------------------------------------------------------------- the producer in front of the layer
def rms_router(h, add, norm_w, eps: float, router_w, h_out=None, stream=None):
    """glmf::rms_q8 (glm_fast.hpp:534) + the router GEMV (glm_fast_path.cu:6925) in one launch: returns (x f32 [n_embd],
    logits f32 [n_expert]); h_out receives h + add when given.  router_w: [n_expert, n_embd] f32 or bf16."""
    n_embd, n_expert = h.numel(), router_w.shape[0]
    assert router_w.dtype in (torch.float32, torch.bfloat16) and router_w.shape[1] == n_embd
    x = torch.empty(n_embd, dtype=torch.float32, device=h.device)
    logits = torch.empty(n_expert, dtype=torch.float32, device=h.device)
    _check("rms_router", _lib.load().maya_rms_router(_ptr(h), _ptr(add), _ptr(norm_w), eps, n_embd, _ptr(router_w),
                                                    int(router_w.dtype == torch.bfloat16), n_expert, _ptr(h_out), _ptr(x),
                                                    _ptr(logits), _stream(stream)))
    return x, logits


def _matrix(t, shape):
    """(address, elements between rows) of a matrix of that shape (one row: [n] too) whose rows are contiguous."""
    strides = t.stride()
    assert t.shape == shape or (shape[0] == 1 and t.shape == shape[1:]), "rows of another shape"
    assert t.dtype is torch.float32 or t.dtype is torch.bfloat16
    assert strides[-1] == 1 or shape[1] <= 1
    return t.data_ptr(), strides[0] if shape[0] > 1 else shape[1]


def xq_bytes(image: int, rows: int, n: int) -> int:
    """Bytes of `rows` 8-bit rows of n values."""
    return (rows * n >> 5) * 36 if image == XQ_Q8_1 else rows * 2 * (n + ((n >> 5) + 63 & ~63))        # (maya_mmq_q8_bytes)


def rms_q8(h, add, norm_w, eps: float, image: int | None = XQ_Q8_1, xq=None, h_out=None, x=None, stream=None):
    """glmf::rms_q8 (glm_fast.hpp:534) for any number of rows: t = h + add (add None: h), x = rms(t) * norm_w, and x in 8 bits.  h and add [T, n] f32 or
    bf16 (one row: [n] too), rows may lie apart.  image: XQ_Q8_1 or XQ_MMQ, what native_quantize_q8_1(x) or mmq_quantize(x) would write, returned as
    uint8 - in `xq` where it is given; None: no 8-bit rows.  h_out (h's type; may be h): receives t; x (f32 or bf16): the normed rows."""
    s = _here("rms_q8", h, add, norm_w, h_out, x, xq, stream=stream)
    shape = h.shape if h.dim() == 2 else h[None].shape
    T, n = shape
    assert norm_w.dtype is torch.float32 and norm_w.shape == shape[1:] and (h_out is None or h_out.dtype is h.dtype)
    if image is not None:
        need = xq_bytes(image, T, n)
        if xq is None:
            xq = h.new_empty(need or 16, dtype=torch.uint8)
        assert xq.numel() * xq.element_size() >= need, "xq is too small"
    else:
        assert xq is None
    hp, ld_h = _matrix(h, shape)
    ap, ld_add = (None, n) if add is None else _matrix(add, shape)
    op, ld_out = (None, n) if h_out is None else _matrix(h_out, shape)
    rows, ld_x = (None, n) if x is None else _matrix(x, shape)
    bf16 = torch.bfloat16
    a = RmsArgs(hp, ap, _ptr(norm_w), op, rows, _ptr(xq), ld_h, ld_add, ld_out, ld_x, T, n, eps, h.dtype is bf16,
                add is not None and add.dtype is bf16, x is not None and x.dtype is bf16, image or 0)
    _check("rms_q8", _lib.load().maya_rms_q8(C.byref(a), s))
    return xq


def q8_read(xq, rows: int, n: int, image: int = XQ_Q8_1, dtype=torch.bfloat16, stream=None):
    """8-bit rows as the values they stand for: (values [rows, n] of dtype bf16 or f32, sums f16 [rows, n / 32] of their groups before rounding)."""
    s = _here("q8_read", xq, stream=stream)
    assert dtype in (torch.float32, torch.bfloat16) and xq.numel() * xq.element_size() >= xq_bytes(image, rows, n)
    values, sums = xq.new_empty((rows, n), dtype=dtype), xq.new_empty((rows, n >> 5), dtype=torch.float16)
    _check("q8_read", _lib.load().maya_q8_read(_ptr(xq), image, rows, n, dtype is torch.bfloat16, values.data_ptr(), sums.data_ptr(), s))
    return values, sums


# ---------------------------------------------------------------- prompt-path grouped GEMM (tensor cores)
def hc_post(block_out, R_old, post, comb, R_new=None, stream=None):
    """glmf::hc_post: R_new [4, n_embd] = block_out * post[d] + comb[d, :] . R_old[:, e] (comb dst-major)."""
    n = block_out.numel()
    R_new = R_new if R_new is not None else torch.empty((4, n), dtype=torch.float32, device=block_out.device)
    _check("hc_post", _lib.load().maya_hc_post(_ptr(block_out), _ptr(R_old), _ptr(post), _ptr(comb), n, _ptr(R_new), _stream(stream)))
    return R_new


def mmq_supported(ggml_type: int) -> bool:
    """mmq::supported (include/strata/prefill/moe_mmq.hpp:16)."""
    return bool(_lib.load().maya_mmq_supported(ggml_type))


def mmq_q8_bytes(rows: int, cols: int) -> int:
    """mmq::q8_bytes (moe_mmq.hpp:20)."""
    return int(_lib.load().maya_mmq_q8_bytes(rows, cols))


def mmq_quantize(x, ids, ggml_type: int, rows: int | None = None, xq=None, stream=None):
    """mmq::quantize (moe_mmq.hpp:34): row i of the result = q8_1 of x[ids[i]] (x[i] when ids is None)."""
    cols, ld = x.shape[1], x.stride(0)
    rows = rows if rows is not None else (ids.numel() if ids is not None else x.shape[0])
    xq = xq if xq is not None else torch.empty(max(mmq_q8_bytes(rows, cols), 16), dtype=torch.uint8, device=x.device)
    assert x.dtype in (torch.float32, torch.bfloat16)
    fn = _lib.load().maya_mmq_quantize_bf16 if x.dtype == torch.bfloat16 else _lib.load().maya_mmq_quantize
    _check("mmq_quantize", fn(_ptr(x), _ptr(ids), _ptr(xq), ggml_type, cols, ld, rows, _stream(stream)))
    return xq


def mmq_quantize_routed(x, pos, k: int, ggml_type: int, xq=None, stream=None):
    """No counterpart in the reference: every row of x rounded once, its q8_1 image stored to the k rows pos[t * k + j]
    (pos from expert_groups) - the bytes mmq_quantize(x, row_tok, ...) writes."""
    assert x.dtype in (torch.float32, torch.bfloat16)
    T, cols, ld = x.shape[0], x.shape[1], x.stride(0)
    xq = xq if xq is not None else torch.empty(max(mmq_q8_bytes(T * k, cols), 16), dtype=torch.uint8, device=x.device)
    fn = _lib.load().maya_mmq_quantize_routed_bf16 if x.dtype == torch.bfloat16 else _lib.load().maya_mmq_quantize_routed
    _check("mmq_quantize_routed", fn(_ptr(x), _ptr(pos), k, _ptr(xq), ggml_type, cols, ld, T, _stream(stream)))
    return xq


def mmq_product(w, ggml_type: int, w_rows: int, w_cols: int, expert_bytes: int, n: int, xq, bounds, ids,
                total_rows: int, dst, ld_dst: int, max_rows: int = 0, expert_map=None, error=None, xq_out=None) -> MmqProduct:
    """mmq::Product (moe_mmq.hpp:41-53).  The tensors must outlive the launch: the struct holds raw addresses."""
    return MmqProduct(_ptr(w), ggml_type, w_rows, w_cols, expert_bytes, n, _ptr(xq), _ptr(bounds), _ptr(ids), total_rows,
                      max_rows, _ptr(dst), ld_dst, _ptr(expert_map), _ptr(error), _ptr(xq_out))


def mmq_run(p: MmqProduct, stream=None) -> None:
    """mmq::Context::run (moe_mmq.hpp:74)."""
    _check("mmq_run", _lib.load().maya_mmq_run(C.byref(p), _stream(stream)))


def mmq_run_glu(p: MmqProduct, limit: float = INF, stream=None) -> None:
    """mmq::Context::run_glu (moe_mmq.hpp:81)."""
    _check("mmq_run_glu", _lib.load().maya_mmq_run_glu(C.byref(p), limit, _stream(stream)))


def mmq_run_chain(gate_up, down, limit: float, counters, stream=None) -> None:
    """No counterpart in the reference: mmq_run_glu of every gate_up product, then mmq_run of every down product (down[i] on
    gate_up[i].xq_out), overlapped where one product's last tiles leave SMs idle.  counters: uint8, zeroed once,
    maya_mmq_chain_bytes long."""
    n = len(gate_up)
    if n == 0:
        return
    _check("mmq_run_chain", _lib.load().maya_mmq_run_chain((MmqProduct * n)(*gate_up), (MmqProduct * n)(*down), n, limit,
                                                           _ptr(counters), counters.numel(), _stream(stream)))


# ---------------------------------------------------------------- whole layer
@dataclass
class MoeLayerConfig:
    n_embd: int
    n_ff: int
    n_expert: int
    k: int
    gu_type: int
    d_type: int
    n_ff_sh: int = 0
    sh_gu_type: int = Q8_0
    sh_d_type: int = Q8_0
    limit: float = INF

    @property
    def blob_bytes(self) -> int:
        return 2 * self.n_ff * row_bytes(self.gu_type, self.n_embd) + self.n_embd * row_bytes(self.d_type, self.n_ff)

    @property
    def shared_bytes(self) -> int:
        if not self.n_ff_sh:
            return 0
        return 2 * self.n_ff_sh * row_bytes(self.sh_gu_type, self.n_embd) + self.n_embd * row_bytes(self.sh_d_type, self.n_ff_sh)


def width_slice(cfg: MoeLayerConfig, experts, shared, lo: int, hi: int, sh_lo: int | None = None, sh_hi: int | None = None):
    """(cfg', experts', shared'): FFN rows lo..hi-1 of every routed expert (sh_lo..sh_hi-1 of the shared one) as blobs
    of their own - each expert's gate and up rows of that range and the same COLUMNS of its down rows.

    A width slice of an expert is an expert of FFN width hi - lo, and the slices' outputs add up to the whole expert's:
    out = sum over slices of down[:, slice] . SwiGLU(gate[slice] x, up[slice] x).  This is how the reference splits
    experts under tensor parallelism (its experts are width-sliced, never partitioned by id): every rank then carries
    1 / N of EVERY token's work whatever the routing, where a partition by expert id gives a rank whatever share of
    the token's experts it happens to hold.  The partial outputs are summed by the same all-reduce.  lo, hi must be
    multiples of the down type's block size (256 for the k- and i-quants) so that the column slice is whole blocks; the
    result is this rank's resident copy (nothing refers to the full blobs afterwards)."""
    H = cfg.n_embd

    def cut(blob, gu_t, d_t, n_ff, a, b):          # blob: [..., blob_bytes]
        rb, drb = row_bytes(gu_t, H), row_bytes(d_t, n_ff)
        gu = n_ff * rb
        lead = blob.shape[:-1]
        gate = blob[..., :gu].reshape(*lead, n_ff, rb)[..., a:b, :].reshape(*lead, -1)
        up = blob[..., gu:2 * gu].reshape(*lead, n_ff, rb)[..., a:b, :].reshape(*lead, -1)
        down = blob[..., 2 * gu:].reshape(*lead, H, drb)[..., row_bytes(d_t, a):row_bytes(d_t, b)].reshape(*lead, -1)
        return torch.cat([gate, up, down], dim=-1).contiguous()

    def whole_blocks(t, *vals):
        for v in vals:
            if v % _BLOCK[t] != 0:
                raise ValueError(f"width slice bound {v} is not a multiple of the block size {_BLOCK[t]}")

    whole_blocks(cfg.d_type, lo, hi)
    ex = cut(experts, cfg.gu_type, cfg.d_type, cfg.n_ff, lo, hi)
    sh, n_ff_sh = None, 0
    if shared is not None and cfg.n_ff_sh:
        sh_lo = lo if sh_lo is None else sh_lo
        sh_hi = hi if sh_hi is None else sh_hi
        whole_blocks(cfg.sh_d_type, sh_lo, sh_hi)
        sh = cut(shared, cfg.sh_gu_type, cfg.sh_d_type, cfg.n_ff_sh, sh_lo, sh_hi)
        n_ff_sh = sh_hi - sh_lo
    out = MoeLayerConfig(cfg.n_embd, hi - lo, cfg.n_expert, cfg.k, cfg.gu_type, cfg.d_type, n_ff_sh, cfg.sh_gu_type,
                         cfg.sh_d_type, cfg.limit)
    return out, ex, sh


class MoeLayer:
    """One resident MoE layer: `experts` uint8 [n_expert, blob_bytes] on the device, optional `shared` blob.

    forward(logits, x) runs route -> experts -> combine for up to 16 tokens and returns (ids, weights, out).
    expert_range = (lo, hi) restricts this rank to experts lo..hi-1 (expert-parallel partition); the others' terms are
    left out of `out` (another rank adds them).  shared_range = (lo, hi) gives this rank a slice of the shared expert's
    FFN width instead of all of it (single-token calls only).  sigmoid = (bias [n_expert] or None, w_scale, norm_w):
    sigmoid routing with a selection bias instead of softmax.  cpu_part [T, n_embd] f32 / cpu_flag [T] i32: a host lane's
    contribution, added to token t's output when cpu_flag[t] != 0 (the tier hooks of the reference's MoeDev).  routing (a GroupRouting): routing over
    groups of experts, a launch of its own in front of the window kernels (no peer, no hc)."""

    def __init__(self, cfg: MoeLayerConfig, experts, shared=None, expert_range=None, shared_here=True, max_tokens: int = 16,
                 staged: bool = False, shared_range=None, sigmoid=None, cpu_part=None, cpu_flag=None, routing: GroupRouting | None = None):
        if routing is not None and (sigmoid is not None or shared_range is not None):
            raise MayaError("moe_layer: routing over groups beside sigmoid or shared_range", -1)
        self.cfg, self.routing = cfg, routing
        self.experts = experts
        self.shared = shared
        lo, hi = expert_range if expert_range is not None else (0, cfg.n_expert)
        self.desc = MoeLayerDesc(cfg.n_embd, cfg.n_ff, cfg.n_expert, cfg.k, cfg.gu_type, cfg.d_type, _ptr(experts),
                                 cfg.blob_bytes, cfg.n_ff_sh if shared is not None else 0, cfg.sh_gu_type,
                                 cfg.sh_d_type, _ptr(shared), cfg.limit, lo, hi, int(bool(shared_here)), int(bool(staged)),
                                 *(shared_range if shared_range is not None else (0, 0)),
                                 *((1, _ptr(sigmoid[0]), float(sigmoid[1]), int(bool(sigmoid[2]))) if sigmoid is not None else (0, None, 1.0, 0)),
                                 _ptr(cpu_part), _ptr(cpu_flag))
        self._keep = (sigmoid, cpu_part, cpu_flag)
        self._ones = {experts.device: self._one(experts.device)}    # not at the first call: a graph's pool that held them would outlive the graph
        self._shapes = {}
        self.max_tokens = max_tokens
        nbytes = int(_lib.load().maya_moe_layer_scratch_bytes(C.byref(self.desc), max_tokens))
        if nbytes == 0:
            raise MayaError("moe_layer_scratch_bytes", -1)
        self.scratch = torch.zeros(nbytes, dtype=torch.uint8, device=experts.device)   # zeroed: holds a barrier counter

    @staticmethod
    def _one(device):
        return torch.empty((), dtype=torch.int32, device=device), torch.empty((), dtype=torch.float32, device=device)

    def _like(self, T, device):
        """What a call's outputs look like (one value of memory each), on the logits' device: torch.empty_like of these takes 1.3 us,
        torch.empty of a shape, a type and a device 2.3."""
        like = self._shapes.get((T, device))
        if like is None:
            i32, f32 = self._ones.get(device) or self._one(device)
            like = (i32.expand(T, self.cfg.k), f32.expand(T, self.cfg.k), f32.expand(T, self.cfg.n_embd))
            if T <= self.max_tokens:             # more are refused: nothing to keep
                self._shapes[T, device] = like
        return like

    def forward(self, logits, x, ids=None, weights=None, out=None, stream=None, peer=None, hc=None):
        """hc = (R_old [T, 4, n_embd], post [T, 4], comb [T, 4, 4], R_new [T, 4, n_embd]): also write the block's output
        into the residual stack (glmf::hc_post) - in the layer kernel's epilogue for one token."""
        T = logits.shape[0]
        if ids is None or weights is None or out is None:
            like = self._like(T, logits.device)
            ids = ids if ids is not None else torch.empty_like(like[0], memory_format=torch.contiguous_format)
            weights = weights if weights is not None else torch.empty_like(like[1], memory_format=torch.contiguous_format)
            out = out if out is not None else torch.empty_like(like[2], memory_format=torch.contiguous_format)
        assert x.dtype in (torch.float32, torch.bfloat16)
        if self.routing is not None:
            if peer is not None or hc is not None:
                raise MayaError("moe_layer: routing over groups with peer or hc", -1)
            assert logits.shape[1] == self.cfg.n_expert and x.shape == (T, self.cfg.n_embd)
            self.routing.route(logits, self.cfg.k, ids, weights, stream)
            return ids, weights, self.forward_routed(ids, weights, x, out, stream)
        if hc is not None:
            args = HcPostArgs(*[_ptr(t) for t in hc])
            seq = 0
            if peer is not None:
                seq = 0 if peer.device_seq else peer.next_seq()
            _check("moe_layer_decode_hc",
                   _lib.load().maya_moe_layer_decode_hc(C.byref(self.desc), _ptr(logits), _ptr(x), int(x.dtype == torch.bfloat16),
                                                        T, _ptr(ids), _ptr(weights), _ptr(out), _ptr(self.scratch),
                                                        self.scratch.numel(), C.byref(peer.desc) if peer is not None else None,
                                                        peer.mi if peer is not None else 0, seq, C.byref(args), _stream(stream)))
            return ids, weights, out
        if peer is not None:     # expert-parallel: `out` becomes the rank-ordered sum over the group (peer.PeerRank)
            _check("moe_layer_decode_ar",
                   _lib.load().maya_moe_layer_decode_ar(C.byref(self.desc), _ptr(logits), _ptr(x), int(x.dtype == torch.bfloat16),
                                                        T, _ptr(ids), _ptr(weights), _ptr(out), _ptr(self.scratch),
                                                        self.scratch.numel(), C.byref(peer.desc), peer.mi,
                                                        0 if peer.device_seq else peer.next_seq(),
                                                        _stream(stream)))
            return ids, weights, out
        _check("moe_layer_decode",
               _lib.load().maya_moe_layer_decode(C.byref(self.desc), _ptr(logits), _ptr(x), int(x.dtype == torch.bfloat16), T,
                                                 _ptr(ids), _ptr(weights), _ptr(out), _ptr(self.scratch),
                                                 self.scratch.numel(), _stream(stream)))
        return ids, weights, out

    def forward_routed(self, ids, weights, x, out=None, stream=None):
        """The layer for up to 16 tokens that are routed already: ids i32 and weights f32 [T, k] (an id outside 0 .. n_expert - 1 contributes nothing)."""
        T, k = ids.shape
        assert k == self.cfg.k and ids.dtype is torch.int32 and weights.dtype is torch.float32 and weights.shape == ids.shape
        assert x.dtype in (torch.float32, torch.bfloat16) and x.shape == (T, self.cfg.n_embd)
        if out is None:
            out = torch.empty((T, self.cfg.n_embd), dtype=torch.float32, device=ids.device)
        assert out.dtype is torch.float32 and out.numel() == T * self.cfg.n_embd
        _check("moe_layer_decode_routed",
               _lib.load().maya_moe_layer_decode_routed(C.byref(self.desc), _ptr(ids), _ptr(weights), _ptr(x), int(x.dtype == torch.bfloat16), T,
                                                        _ptr(out), _ptr(self.scratch), self.scratch.numel(), _stream(stream)))
        return out

    def forward_checked(self, logits, x, kernel: int, polls: int = 1 << 22, out=None, hc=None, stream=None):
        """forward of one token (not of a layer with routing over groups) with the caller's choice of kernel (LAYER_CHOICE, LAYER_FUSED, LAYER_TOKEN, LAYER_STAGED; a kernel that
        does not take the layer raises) and bound on its waits for weight rows."""
        if self.routing is not None:
            raise MayaError("moe_layer: routing over groups runs the window kernels", -1)
        dev = logits.device
        ids = torch.empty((1, self.cfg.k), dtype=torch.int32, device=dev)
        weights = torch.empty((1, self.cfg.k), dtype=torch.float32, device=dev)
        out = out if out is not None else torch.empty((1, self.cfg.n_embd), dtype=torch.float32, device=dev)
        assert logits.shape[0] == 1 and x.dtype in (torch.float32, torch.bfloat16)
        args = C.byref(HcPostArgs(*[_ptr(t) for t in hc])) if hc is not None else None
        _check("moe_layer_decode_checked",
               _lib.load().maya_moe_layer_decode_checked(C.byref(self.desc), _ptr(logits), _ptr(x), int(x.dtype == torch.bfloat16),
                                                         _ptr(ids), _ptr(weights), _ptr(out), _ptr(self.scratch), self.scratch.numel(),
                                                         kernel, polls, args, _stream(stream)))
        return ids, weights, out

    def phase_ns(self, stream=None):
        """Block 0's phase stamps of the last single-token launch (fused or token kernel), as offsets in ns from its start."""
        buf = (C.c_ulonglong * 6)()
        _check("moe_layer_phase_ns", _lib.load().maya_moe_layer_phase_ns(C.byref(self.desc), _ptr(self.scratch), _stream(stream), buf))
        return [int(buf[i]) - int(buf[0]) for i in range(6)]

    def error(self, stream=None) -> int:
        """The scratch's sticky device-side error word (0 = none); synchronises the stream."""
        return int(_lib.load().maya_moe_layer_error(C.byref(self.desc), self.max_tokens, _ptr(self.scratch), _stream(stream)))


class MoePrefill:
    """The prompt path of one resident layer for a chunk of up to `max_tokens` tokens, with no host round trip:
    route -> group rows by expert -> each token rounded to q8_1 once and stored to its k sorted rows -> one chain of grouped
    GEMMs (gate/up with SwiGLU and the q8_1 rounding of h in its write-back, then down; every pool's products and, over all
    rows, the shared expert's) -> weighted combine.

    Follows the reference's prefill_run expert sequence (src/core/glm_prefill.cu:3230-3420: expert_count, bases,
    expert_scatter, mmq::quantize, Context::run_glu, mmq::quantize, Context::run, moe_combine), except that the bases
    are scanned on the device.  Every buffer is allocated once, here.

    expert_range = (lo, hi) makes this an expert-parallel rank: only experts lo..hi-1 are multiplied and combined, and
    the returned ffn is this rank's partial sum (the ranks' results add up; pass `shared` on one rank only).

    `experts` is uint8 [n_expert, blob_bytes] of one type (cfg.gu_type == cfg.d_type is not required), or None with
    `pools` = [(ggml_type, blobs uint8 [n_i, blob_bytes of that type], expert ids of the n_i blobs), ...] for a layer whose
    experts are stored in different types: one product per pool, each matrix finding its rows through the pool's
    expert map (the reference's staged groups, moe_mmq.hpp:41-53 with bounds per group).

    routing (a GroupRouting): routing over groups of experts instead of the softmax top-k."""

    def __init__(self, cfg: MoeLayerConfig, experts, shared=None, max_tokens: int = 4096, pools=None, expert_range=None,
                 routing: GroupRouting | None = None):
        self.routing = routing
        H, FF = cfg.n_embd, cfg.n_ff
        self.expert_range = expert_range         # (lo, hi): an expert-parallel rank's experts; ffn is then its partial sum
        if pools is None:
            if expert_range is None:
                pools = [((cfg.gu_type, cfg.d_type), experts, None)]
            else:                                # this rank's blobs only (a view), found through an expert map
                lo, hi = expert_range
                pools = [((cfg.gu_type, cfg.d_type), experts[lo:hi], list(range(lo, hi)))] if hi > lo else []
        elif expert_range is not None:
            lo, hi = expert_range
            kept = []
            for types, blobs, expert_ids in pools:
                sel = [i for i, e in enumerate(expert_ids) if lo <= e < hi]
                if sel:
                    kept.append((types, blobs[sel[0]:sel[-1] + 1] if sel == list(range(sel[0], sel[-1] + 1)) else blobs[sel].contiguous(),
                                 [expert_ids[i] for i in sel]))
            pools = kept
        self.pools = []
        for types, blobs, expert_ids in pools:
            gt, dt = types if isinstance(types, tuple) else (types, types)
            if not (mmq_supported(gt) and mmq_supported(dt)):
                raise MayaError("MoePrefill: type without a grouped GEMM", -2)
            stride = 2 * FF * row_bytes(gt, H) + H * row_bytes(dt, FF)
            assert blobs.shape[1] == stride, "a pool's blobs must be [gate | up | down] of its own type"
            emap = None if expert_ids is None else torch.as_tensor(expert_ids, dtype=torch.int32).to(blobs.device)
            self.pools.append((gt, dt, blobs, stride, 2 * FF * row_bytes(gt, H), blobs.shape[0], emap))
        if shared is not None and not (mmq_supported(cfg.sh_gu_type) and mmq_supported(cfg.sh_d_type)):
            raise MayaError("MoePrefill: shared expert's type without a grouped GEMM", -2)
        self.cfg, self.shared, self.max_tokens = cfg, shared, max_tokens
        dev, T, k, E = (self.pools[0][2].device if self.pools else experts.device), max_tokens, cfg.k, cfg.n_expert
        i32 = dict(dtype=torch.int32, device=dev)
        f32 = dict(dtype=torch.float32, device=dev)
        u8 = dict(dtype=torch.uint8, device=dev)
        n = T * k
        self.ids, self.weights = torch.empty((T, k), **i32), torch.empty((T, k), **f32)
        self.counts, self.rank, self.bounds = torch.empty(E, **i32), torch.empty(n, **i32), torch.empty(E + 1, **i32)
        self.pos, self.row_tok = torch.empty(n, **i32), torch.empty(n, **i32)
        self.xq = torch.empty(mmq_q8_bytes(n, H), **u8)
        self.hq = torch.empty(mmq_q8_bytes(n, FF), **u8)
        self.out, self.ffn = torch.empty((n, H), **f32), torch.empty((T, H), **f32)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        chain_bytes = _lib.load().maya_mmq_chain_bytes
        self.chain = torch.zeros(chain_bytes(n, sum(p[5] for p in self.pools) + 1, len(self.pools) + 1), **u8)      # + the shared expert
        if shared is not None:
            FS = cfg.n_ff_sh
            self.sh_bounds, self._sh_T = torch.zeros(2, **i32), -1
            self.sh_xq = torch.empty(mmq_q8_bytes(T, H), **u8)
            self.sh_hq = torch.empty(mmq_q8_bytes(T, FS), **u8)
            self.sh_out = torch.empty((T, H), **f32)
            self.sh_down_off = 2 * FS * row_bytes(cfg.sh_gu_type, H)

    def forward(self, logits, x, stream=None, peer=None):
        """peer (a peer.PeerRank whose stride holds T * n_embd floats), on an expert-parallel rank: the returned ffn is the
        rank-ordered sum over the group, exchanged inside the combine launch."""
        cfg, lib, s = self.cfg, _lib.load(), _stream(stream)
        T, k, H, FF, E = logits.shape[0], cfg.k, cfg.n_embd, cfg.n_ff, cfg.n_expert
        assert T <= self.max_tokens and x.shape == (T, H) and x.dtype in (torch.float32, torch.bfloat16)
        n = T * k
        quant = lib.maya_mmq_quantize_bf16 if x.dtype == torch.bfloat16 else lib.maya_mmq_quantize
        quant_routed = lib.maya_mmq_quantize_routed_bf16 if x.dtype == torch.bfloat16 else lib.maya_mmq_quantize_routed
        ids, w = self.ids[:T], self.weights[:T]
        if self.routing is None:
            _check("router_top10", lib.maya_router_top10(_ptr(logits), T, E, k, _ptr(ids), _ptr(w), s))
        else:
            assert logits.shape == (T, E)
            self.routing.route(logits, k, ids, w, s)
        if n <= 4096 and E <= 1024:  # one block does it all: 20 tokens of top 8 109.6 / 107.0 us a layer, 300 135.9 / 134.3; 2000 over 512 experts 457 / 466
            _check("expert_group", lib.maya_expert_group_counts(_ptr(ids), n, k, E, _ptr(self.counts), _ptr(self.rank), _ptr(self.bounds),
                                                                _ptr(self.row_tok), _ptr(self.pos), s))
        else:
            _check("expert_count", lib.maya_expert_count(_ptr(ids), n, E, _ptr(self.counts), _ptr(self.rank), s))
            _check("expert_bounds", lib.maya_expert_bounds(_ptr(self.counts), E, _ptr(self.bounds), s))
            _check("expert_scatter", lib.maya_expert_scatter(_ptr(ids), _ptr(self.rank), _ptr(self.bounds), n, k,
                                                             _ptr(self.row_tok), _ptr(self.pos), s))
        qtype = self.pools[0][0] if self.pools else cfg.gu_type
        # each token rounded once, its image stored to its k sorted rows (the bytes quant(x, row_tok, ...) would write)
        _check("mmq_quantize_routed", quant_routed(_ptr(x), _ptr(self.pos), k, _ptr(self.xq), qtype, H, x.stride(0), T, s))
        # h leaves the gate/up products already quantized
        gu = [mmq_product(blobs, gt, 2 * FF, H, stride, n_p, self.xq, self.bounds, None, n, None, FF, expert_map=emap,
                          error=self.err, xq_out=self.hq) for gt, dt, blobs, stride, down_off, n_p, emap in self.pools]
        dn = [mmq_product(blobs.data_ptr() + down_off, dt, H, FF, stride, n_p, self.hq, self.bounds, None, n, self.out, H,
                          expert_map=emap, error=self.err) for gt, dt, blobs, stride, down_off, n_p, emap in self.pools]
        sh_out = None
        if self.shared is not None:  # one more pair of products, in the same chain
            FS = cfg.n_ff_sh
            if self._sh_T != T:      # the shared expert is one more "expert" that owns every row
                self.sh_bounds[1], self._sh_T = T, T
            _check("mmq_quantize", quant(_ptr(x), None, _ptr(self.sh_xq), cfg.sh_gu_type, H, x.stride(0), T, s))
            gu.append(mmq_product(self.shared, cfg.sh_gu_type, 2 * FS, H, cfg.shared_bytes, 1, self.sh_xq, self.sh_bounds, None, T,
                                  None, FS, error=self.err, xq_out=self.sh_hq))
            dn.append(mmq_product(self.shared.data_ptr() + self.sh_down_off, cfg.sh_d_type, H, FS, cfg.shared_bytes, 1, self.sh_hq,
                                  self.sh_bounds, None, T, self.sh_out, H, error=self.err))
            sh_out = self.sh_out
        mmq_run_chain(gu, dn, cfg.limit, self.chain, s)
        ffn = self.ffn[:T]
        if self.expert_range is None:
            _check("moe_combine_rows", lib.maya_moe_combine_rows(_ptr(self.out), _ptr(self.pos), _ptr(w), _ptr(sh_out), T, k, H,
                                                                _ptr(ffn), s))
        elif peer is not None:
            _check("moe_combine_rows_local_ar",
                   lib.maya_moe_combine_rows_local_ar(_ptr(self.out), _ptr(self.pos), _ptr(w), _ptr(ids), self.expert_range[0],
                                                      self.expert_range[1], _ptr(sh_out), T, k, H, _ptr(ffn), C.byref(peer.desc),
                                                      peer.mi, 0 if peer.device_seq else peer.next_seq(), s))
        else:
            _check("moe_combine_rows_local",
                   lib.maya_moe_combine_rows_local(_ptr(self.out), _ptr(self.pos), _ptr(w), _ptr(ids), self.expert_range[0],
                                                   self.expert_range[1], _ptr(sh_out), T, k, H, _ptr(ffn), s))
        return ids, w, ffn

    def error(self) -> int:
        """1 when a bounded wait inside a grouped-GEMM launch ran out (synchronises; sticky).  A chain that ended that way leaves its
        counters somewhere in between, and the next one would start from there: they are zeroed here, so that the passes after
        this call are sound again."""
        code = int(self.err.item())
        if code:
            self.chain.zero_()
        return code


# ---------------------------------------------------------------- attention over a paged 8-bit cache
KV_BLOCK = 64                # tokens of a block (MAYA_KV_BLOCK)


class KvCache:
    """The keys and values of a layer's sequences in 8 bits: blocks of 64 tokens with an f32 scale a block and key/value head
    (include/maya_attn.h states the layout).  A handle over the caller's tensors; KvCache.empty allocates them.

    k uint8 [n_blocks, n_kv, head_dim / 64, 64, 64] (the last two: token, value), v uint8 [n_blocks, n_kv, head_dim, 64], k_scale and
    v_scale f32 [n_blocks, n_kv], table i32 [n_seq, blocks of a sequence] (which block holds tokens 64 b .. of sequence s), k_sum
    int16 [n_blocks, n_kv, head_dim] or None (block selection needs it).  Entries of `table` may be changed between calls; where its
    first dimension is longer than a batch, the batch's sequences are its first rows."""

    def __init__(self, k, v, k_scale, v_scale, table, k_sum=None):
        n_blocks, n_kv, panels, tokens, width = k.shape
        head_dim = 64 * panels
        assert (tokens, width) == (KV_BLOCK, 64) and v.shape == (n_blocks, n_kv, head_dim, KV_BLOCK) and table.dim() == 2
        assert k_scale.shape == v_scale.shape == (n_blocks, n_kv) and (k_sum is None or k_sum.shape == (n_blocks, n_kv, head_dim))
        assert k.dtype == v.dtype == torch.uint8 and k_scale.dtype == v_scale.dtype == torch.float32 and table.dtype == torch.int32
        assert k_sum is None or k_sum.dtype == torch.int16
        self.k, self.v, self.k_scale, self.v_scale, self.table, self.k_sum = k, v, k_scale, v_scale, table, k_sum
        self.n_blocks, self.n_kv, self.head_dim, self.n_seq = n_blocks, n_kv, head_dim, table.shape[0]
        self.block_values = KV_BLOCK * n_kv * head_dim
        self.desc = KvCacheDesc(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), _ptr(k_sum), _ptr(table), table.shape[1], n_blocks, n_kv,
                                head_dim)
        self._ref = C.byref(self.desc)

    @classmethod
    def empty(cls, n_blocks: int, n_kv: int, head_dim: int, table, sums: bool = True):
        """A cache of n_blocks blocks on the table's device; its contents are whatever the memory held."""
        dev = table.device
        return cls(torch.empty((n_blocks, n_kv, head_dim // 64, KV_BLOCK, 64), dtype=torch.uint8, device=dev),
                   torch.empty((n_blocks, n_kv, head_dim, KV_BLOCK), dtype=torch.uint8, device=dev),
                   torch.empty((n_blocks, n_kv), dtype=torch.float32, device=dev), torch.empty((n_blocks, n_kv), dtype=torch.float32, device=dev),
                   table, torch.empty((n_blocks, n_kv, head_dim), dtype=torch.int16, device=dev) if sums else None)

    def read(self, blocks, counts=None, k=None, v=None, mean=None, dtype=torch.bfloat16, stream=None):
        """Blocks (i32 [n]) as the values they stand for: k and v [n, 64, n_kv, head_dim], and the mean key [n, n_kv, head_dim] of each
        block's first counts[i] tokens (None without sums); tokens from counts[i] on are zeros."""
        n, dev = blocks.numel(), blocks.device
        if k is None:
            k = torch.empty((n, KV_BLOCK, self.n_kv, self.head_dim), dtype=dtype, device=dev)
        if v is None:
            v = torch.empty((n, KV_BLOCK, self.n_kv, self.head_dim), dtype=dtype, device=dev)
        if mean is None and self.k_sum is not None:
            mean = torch.empty((n, self.n_kv, self.head_dim), dtype=dtype, device=dev)
        assert k.dtype == v.dtype and (mean is None or mean.dtype == k.dtype) and k.dtype in (torch.float32, torch.bfloat16)
        assert k.numel() == v.numel() == n * self.block_values and (mean is None or mean.numel() == n * self.block_values // KV_BLOCK)
        assert blocks.dtype == torch.int32 and (counts is None or (counts.dtype == torch.int32 and counts.numel() == n))
        _check("kv_read", _lib.load().maya_kv_read(self._ref, _ptr(blocks), _ptr(counts), n, int(k.dtype == torch.bfloat16), _ptr(k), _ptr(v),
                                                   _ptr(mean), _stream(stream)))
        return k, v, mean


class AttnBatch:
    """The new tokens of a pass: those of sequence s are rows start[s] .. start[s + 1] - 1 (i32 [n_seq + 1]) and the last of its
    kv_len[s] tokens (i32 [n_seq]; it counts them).  n_tokens = start[n_seq]; max_new and max_len: upper bounds of the new tokens and
    of kv_len of any sequence, which size the launches; min_len: a lower bound of kv_len of those that have new tokens."""

    def __init__(self, start, kv_len, n_tokens: int, max_new: int, max_len: int, min_len: int = 0):
        assert start.dtype == kv_len.dtype == torch.int32 and start.numel() == kv_len.numel() + 1
        self.start, self.kv_len, self.n_tokens, self.n_seq, self.min_len = start, kv_len, n_tokens, kv_len.numel(), min_len
        self.desc = AttnBatchDesc(_ptr(start), _ptr(kv_len), kv_len.numel(), n_tokens, max_new, max_len)
        self._ref = C.byref(self.desc)

    @classmethod
    def of(cls, new, kv_len, device="cuda"):
        """From host lists: the new tokens of every sequence and its tokens with them."""
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        return cls(torch.tensor(start, dtype=torch.int32, device=device), torch.tensor(list(kv_len), dtype=torch.int32, device=device),
                   start[-1], max(new, default=0), max(kv_len, default=0), min((n for m, n in zip(new, kv_len) if m), default=0))


class KvPages:
    """The blocks of one or more layers' caches (KvCaches over one table, of one shape), handed out, shared and taken back on the device: nothing here
    waits for the GPU, and captured calls do in a replay what they would then do.  refs i32 [n_blocks]: how many entries of the table hold a block (0: free; None:
    counted from the table here).  Table entries without a block are -1.  A call that needs blocks gets the free ones of the lowest numbers, of those that are
    free when it begins; too few leave -1 behind, and error() says so: a sequence with -1 in front of its length has lost the tokens of that block - free it and prefill
    it again.  One thread and one stream at a time (include/maya_attn.h)."""

    def __init__(self, caches, refs=None):
        first = caches[0]
        shape = lambda c: (c.table.data_ptr(), c.table.shape, c.n_blocks, c.n_kv, c.head_dim, c.k_sum is None, c.k.device)   # noqa: E731
        assert all(shape(c) == shape(first) for c in caches), "caches of one table and one shape expected"
        dev, table = first.k.device, first.table
        assert all(t is None or t.device == dev for c in caches for t in (c.v, c.k_scale, c.v_scale, c.table, c.k_sum)), "caches on one device expected"
        if refs is None:
            held = table[(table >= 0) & (table < first.n_blocks)].long()
            refs = torch.bincount(held, minlength=first.n_blocks).to(torch.int32)
        assert refs.dtype is torch.int32 and refs.shape == (first.n_blocks,) and refs.device == dev and table.device == dev
        self.caches, self.table, self.refs = list(caches), table, refs
        self.n_blocks, self.n_seq = first.n_blocks, table.shape[0]
        self._layers = torch.tensor([[0 if t is None else t.data_ptr() for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_sum)] for c in caches],
                                    dtype=torch.int64).to(dev)
        self.desc = KvPagesDesc(_ptr(self._layers), _ptr(table), _ptr(refs), None, 0, table.shape[0], table.shape[1], first.n_blocks, len(caches), first.n_kv,
                                first.head_dim, int(first.k_sum is not None))
        nbytes = int(_lib.load().maya_pages_scratch_bytes(C.byref(self.desc)))
        if nbytes == 0:
            raise MayaError("pages_scratch_bytes", -1)
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.scratch[:256].zero_()
        self.desc.scratch, self.desc.scratch_bytes = self.scratch.data_ptr(), nbytes
        self.live = self.scratch[8:12].view(torch.int32)     # i32 [1]: live blocks as the last compact() found them
        self._ref = C.byref(self.desc)

    def _list(self, what, stream, *lists):
        s = _here(what, self.scratch, *lists, stream=stream)
        n = lists[0].numel()
        for t in lists:
            assert t.dtype is torch.int32 and t.numel() == n
        return n, s, *map(_ptr, lists)

    def reserve(self, batch: AttnBatch, stream=None) -> None:
        """Blocks for the batch's new tokens, in front of append(): entries without one get one, a block that other sequences hold too is replaced by a
        block of the sequence's own (with a copy of the tokens from before in it)."""
        s = _here("pages_reserve", self.scratch, batch.start, batch.kv_len, stream=stream)
        _check("pages_reserve", _lib.load().maya_pages_reserve(self._ref, batch._ref, s))

    def fork(self, parents, children, lens, stream=None) -> None:
        """i32 [n] each: sequence children[i] becomes the first lens[i] tokens of sequence parents[i], all at once (a beam search's step).  Full blocks are
        shared, one that is not full is copied; what the children held is given up.  A child that is its own parent is left as it is."""
        n, s, p, c, k = self._list("pages_fork", stream, parents, children, lens)
        _check("pages_fork", _lib.load().maya_pages_fork(self._ref, p, c, k, n, s))

    def free(self, seqs, stream=None) -> None:
        """Sequences seqs (i32 [n]) give up their blocks; their table rows are -1."""
        n, s, q = self._list("pages_free", stream, seqs)
        _check("pages_free", _lib.load().maya_pages_free(self._ref, q, n, s))

    def compact(self, most: int | None = None, stream=None) -> None:
        """The live blocks move to the lowest numbers, tables and counts with them: all that lie too high, or the `most` lowest of these (the next call
        goes on).  `live` says how many blocks are live."""
        s = _here("pages_compact", self.scratch, stream=stream)
        _check("pages_compact", _lib.load().maya_pages_compact(self._ref, self.n_blocks if most is None else most, s))

    def copy(self, src, dst, stream=None) -> None:
        """Blocks src[i] to blocks dst[i] (i32 [n]) in all layers.  No block twice in dst, none in both."""
        n, s, a, d = self._list("pages_copy", stream, src, dst)
        _check("pages_copy", _lib.load().maya_pages_copy(self._ref, a, d, n, s))

    def error(self, stream=None) -> int:
        """1 after a call that found too few free blocks (synchronises the stream); the word is zeroed then."""
        code = int(_lib.load().maya_pages_error(self._ref, _stream(stream)))
        if code < 0:
            raise MayaError("pages_error", code)
        if code > 0:
            self.scratch[:4].zero_()
            torch.cuda.current_stream(self.scratch.device).synchronize()      # (the next call may be on another stream)
        return code


class Rope:
    """What stands between a layer's projections and its attention: cos and sin f32 [positions, rot_dim / 2] (None: no rotation), the
    weights f32 [head_dim] of the queries' and keys' RMS norms (None: no norm).  pairs: value 2 i turns with 2 i + 1, else i with
    i + rot_dim / 2.  Never written after this: layers and threads may share one."""

    def __init__(self, cos=None, sin=None, q_w=None, k_w=None, eps: float = 1e-6, pairs: bool = False):
        for t in (cos, sin, q_w, k_w):
            assert t is None or t.dtype == torch.float32
        assert (cos is None) == (sin is None) and (cos is None or cos.shape == sin.shape)
        n_pos, rot_dim = (cos.shape[0], 2 * cos.shape[1]) if cos is not None else (0, 0)
        self._keep = cos, sin, q_w, k_w
        sizes = {t.numel() for t in (q_w, k_w) if t is not None}
        assert len(sizes) < 2, "norm weights of two head sizes"
        self.head_dim = sizes.pop() if sizes else None       # that the weights are for
        self.args = RopeArgs(q_w=_ptr(q_w), k_w=_ptr(k_w), eps=eps, cos=_ptr(cos), sin=_ptr(sin), n_pos=n_pos, rot_dim=rot_dim, pairs=int(pairs))
        self.image = bytes(self.args)                       # what a call starts from


def _rows(x, n: int, heads: int, head_dim: int):
    """(address, elements between rows) of [n, heads, head_dim] whose heads lie side by side: a view into wider rows is fine."""
    row, head, one = x.stride()
    assert x.is_cuda and x.shape == (n, heads, head_dim) and one == 1 and (heads == 1 or head == head_dim)
    return x.data_ptr(), row if n > 1 else heads * head_dim


class KvAttention:
    """The attention of one layer over a KvCache: n_q query heads, the first n_q / n_kv of which share key/value head 0, and so on.

    append(batch, q, k, v, rope) normalises and rotates the new tokens' queries and keys and puts keys and values into the cache;
    forward(batch, q) attends over it; select(batch, q) chooses the n_sel blocks each token reads and forward(batch, q, sel=...) attends over those
    alone.  f32 or bf16; q, k, v [n_tokens, heads, head_dim], views into rows of projections among them.  scale: of the scores
    (head_dim ** -0.5); window > 0: a token sees the last `window` positions.  Prompt chunks and single tokens at long contexts are better passed as
    two batches (include/maya_attn.h says why).  max_tokens > 0 does not size anything: the scratch is the same for any batch.  The scratch and the arguments of a call belong to this object: one
    thread and one stream at a time."""

    def __init__(self, cache: KvCache, n_q: int, scale: float | None = None, window: int = 0, n_sel: int = 0, n_first: int = 1,
                 n_last: int = 2, max_tokens: int = 65536):
        self.cache, self.n_q, self.n_sel = cache, n_q, n_sel
        nbytes = int(_lib.load().maya_attn_scratch_bytes(cache._ref, n_q, max_tokens))
        if nbytes == 0:
            raise MayaError("attn_scratch_bytes", -1)
        self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=cache.k.device)
        self.scratch[:1 << 12].zero_()                      # the error word and the counters
        self._attn = AttnArgs(None, 0, 0, n_q, cache.head_dim ** -0.5 if scale is None else scale, window, None, 0, None, None)
        self._select = SelectArgs(None, 0, 0, n_q, n_first, n_last, n_sel, None)
        self._rope = RopeArgs()
        self._rope_bytes = memoryview(self._rope).cast("B")
        self._refs = C.byref(self._attn), C.byref(self._select), C.byref(self._rope)

    def _queries(self, a, batch, q):
        """The queries of a call into its arguments; returns their type."""
        dtype, c = q.dtype, self.cache
        assert dtype is torch.float32 or dtype is torch.bfloat16
        assert batch.n_seq <= c.n_seq
        a.is_bf16 = dtype is torch.bfloat16
        a.q, a.ld_q = _rows(q, batch.n_tokens, self.n_q, c.head_dim)
        return dtype

    def append(self, batch: AttnBatch, q, k, v, rope: Rope, pos=None, q_out=None, stream=None):
        """Returns the normalised and rotated queries.  k and v None: queries only.  pos i32 [n_tokens]: rows of cos and sin to turn by
        (None: the tokens' positions)."""
        a, c, n = self._rope, self.cache, batch.n_tokens
        assert rope.head_dim is None or rope.head_dim == c.head_dim, "norm weights [head_dim] expected"
        self._rope_bytes[:] = rope.image
        dtype = self._queries(a, batch, q)
        a.n_q = self.n_q
        if k is not None:
            assert k.dtype is dtype and v.dtype is dtype
            a.k, a.ld_k = _rows(k, n, c.n_kv, c.head_dim)
            a.v, a.ld_v = _rows(v, n, c.n_kv, c.head_dim)
        if q_out is None:
            q_out = torch.empty((n, self.n_q, c.head_dim), dtype=dtype, device=q.device)
        assert q_out.dtype is dtype and q_out.shape == (n, self.n_q, c.head_dim) and (pos is None or (pos.dtype == torch.int32 and pos.numel() == n))
        a.pos, a.q_out = _ptr(pos), _ptr(q_out)
        _check("qk_norm_rope_append", _lib.load().maya_qk_norm_rope_append(c._ref, batch._ref, self._refs[2], _stream(stream)))
        return q_out

    def forward(self, batch: AttnBatch, q, sel=None, out=None, lse=None, stream=None):
        """out [n_tokens, n_q, head_dim] of q's type.  sel i32 [n_tokens, n_kv, n_sel] (select's): the blocks each token reads.
        lse f32 [n_tokens, n_q]: ln of the sum of exp(scores), for joining with attention over other tokens."""
        a, c = self._attn, self.cache
        dtype = self._queries(a, batch, q)
        if out is None:
            out = torch.empty((batch.n_tokens, self.n_q, c.head_dim), dtype=dtype, device=q.device)
        assert out.dtype is dtype and out.shape == (batch.n_tokens, self.n_q, c.head_dim)
        assert lse is None or (lse.dtype == torch.float32 and lse.shape == (batch.n_tokens, self.n_q))
        if sel is not None:
            assert sel.dtype == torch.int32 and sel.shape[:2] == (batch.n_tokens, c.n_kv)
            a.n_sel = sel.shape[2]
        a.sel, a.out, a.lse = _ptr(sel), _ptr(out), _ptr(lse)
        _check("attn_q8", _lib.load().maya_attn_q8(c._ref, batch._ref, self._refs[0], self.scratch.data_ptr(), self.scratch.numel(), _stream(stream)))
        return out

    def select(self, batch: AttnBatch, q, sel=None, stream=None):
        """i32 [n_tokens, n_kv, n_sel]: the blocks each token reads, ascending, -1 behind the last."""
        a, c = self._select, self.cache
        self._queries(a, batch, q)
        if sel is None:
            sel = torch.empty((batch.n_tokens, c.n_kv, self.n_sel), dtype=torch.int32, device=q.device)
        assert sel.dtype == torch.int32 and sel.shape == (batch.n_tokens, c.n_kv, self.n_sel)
        a.sel = _ptr(sel)
        _check("block_select", _lib.load().maya_block_select(c._ref, batch._ref, self._refs[1], _stream(stream)))
        return sel

    def error(self, stream=None) -> int:
        """1 after a call whose bounded wait ran out (its outputs are not valid, and neither are those of the calls since); synchronises the
        stream.  The error word and the counters are zeroed then, so that the calls after this are sound again."""
        code = int(_lib.load().maya_attn_error(self.scratch.data_ptr(), _stream(stream)))
        if code > 0:
            self.scratch[:1 << 12].zero_()
            if self.scratch.is_cuda:
                torch.cuda.current_stream(self.scratch.device).synchronize()      # (the next call may be on another stream)
        return code
