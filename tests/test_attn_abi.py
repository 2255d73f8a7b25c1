"""The attention entry points on a machine without a GPU: sizes and refusals (argument checks come before any launch)."""
import ctypes as C

import pytest


@pytest.fixture
def made():
    from project_maya_b200 import _lib as L
    cache = L.KvCacheDesc(256, 256, 256, 256, 256, 256, 4, 10, 2, 128)
    batch = L.AttnBatchDesc(256, 256, 3, 5, 2, 200)
    rope = L.RopeArgs(q=256, k=256, v=256, ld_q=1024, ld_k=256, ld_v=256, is_bf16=0, n_q=8, eps=1e-6, cos=256, sin=256, n_pos=256, rot_dim=128, q_out=512)
    attn = L.AttnArgs(q=256, ld_q=1024, n_q=8, scale=0.1, out=256)
    sel = L.SelectArgs(q=256, ld_q=1024, n_q=8, n_first=1, n_last=2, n_sel=8, sel=256)
    return L.load(), cache, batch, rope, attn, sel


def calls(lib, cache, batch, rope, attn, sel):
    size = lib.maya_attn_scratch_bytes(C.byref(cache), 8, 1) or 1 << 30
    return {"append": lambda: lib.maya_qk_norm_rope_append(C.byref(cache), C.byref(batch), C.byref(rope), None),
            "attn": lambda: lib.maya_attn_q8(C.byref(cache), C.byref(batch), C.byref(attn), 256, size, None),
            "select": lambda: lib.maya_block_select(C.byref(cache), C.byref(batch), C.byref(sel), None),
            "read": lambda: lib.maya_kv_read(C.byref(cache), 256, None, 3, 0, 256, 256, None, None)}


def test_scratch_size(made):
    lib, cache, *_ = made
    size = lib.maya_attn_scratch_bytes(C.byref(cache), 8, 100)
    assert 0 < size < 100 << 20
    assert lib.maya_attn_scratch_bytes(C.byref(cache), 7, 100) == 0 and lib.maya_attn_scratch_bytes(C.byref(cache), 8, 0) == 0
    cache.head_dim = 96
    assert lib.maya_attn_scratch_bytes(C.byref(cache), 8, 100) == 0


@pytest.mark.parametrize("field,value,status", [("k", None, -1), ("v", 8, -1), ("k_scale", None, -1), ("table", None, -1), ("table_ld", 0, -1), ("n_blocks", 0, -1),
                                                ("n_kv", 0, -1), ("head_dim", 96, -4), ("head_dim", 320, -4), ("k_sum", 8, -1)])
def test_cache_refusals(made, field, value, status):
    lib, cache, *_ = made
    setattr(cache, field, value)
    for name, call in calls(*made).items():
        assert call() == status, name


@pytest.mark.parametrize("field,value,status", [("start", None, -1), ("kv_len", None, -1), ("n_seq", -1, -1), ("n_seq", 0, -1), ("n_tokens", -1, -1), ("n_tokens", 7, -1),
                                                ("max_new", 0, -1), ("max_new", 6, -1), ("max_len", 257, -1), ("max_len", -1, -1), ("n_seq", 70000, -4)])
def test_batch_refusals(made, field, value, status):
    lib, cache, batch, *_ = made
    setattr(batch, field, value)
    for name, call in calls(*made).items():
        assert name == "read" or call() == status, name


@pytest.mark.parametrize("which,field,value,status", [
    ("append", "q", None, -1), ("append", "q_out", None, -1), ("append", "v", None, -1), ("append", "ld_q", 1023, -1), ("append", "ld_k", 255, -1),
    ("append", "rot_dim", 127, -1), ("append", "rot_dim", 130, -1), ("append", "rot_dim", -2, -1), ("append", "cos", None, -1), ("append", "n_pos", 0, -1), ("append", "eps", -1.0, -1),
    ("append", "n_q", 0, -1), ("attn", "q", None, -1), ("attn", "out", None, -1), ("attn", "out", 264, -1), ("attn", "n_q", 7, -1), ("attn", "scale", 0.0, -1),
    ("attn", "scale", -1.0, -1), ("attn", "window", -1, -1), ("attn", "ld_q", 1000, -1), ("select", "q", None, -1), ("select", "sel", None, -1), ("select", "n_q", 5, -1),
    ("select", "n_first", -1, -1), ("select", "n_last", 0, -1), ("select", "n_sel", 2, -1), ("select", "n_sel", 600, -4)])
def test_argument_refusals(made, which, field, value, status):
    from project_maya_b200 import _lib
    lib, cache, batch, rope, attn, sel = made
    setattr({"append": rope, "attn": attn, "select": sel}[which], field, value)
    errors, launches = _lib.load().maya_launch_errors(), _lib.load().maya_launch_count()
    assert calls(*made)[which]() == status
    assert _lib.load().maya_launch_errors() == errors + 1 and _lib.load().maya_launch_count() == launches


def test_other_refusals(made):
    lib, cache, batch, rope, attn, sel = made
    size = lib.maya_attn_scratch_bytes(C.byref(cache), 8, 1)
    for scratch, n in ((None, size), (264, size), (256, size - 1)):            # none, not on 256 bytes, too small
        assert lib.maya_attn_q8(C.byref(cache), C.byref(batch), C.byref(attn), scratch, n, None) == -1
    attn.sel, attn.n_sel = 256, 0
    assert calls(*made)["attn"]() == -1
    attn.n_sel = 513
    assert calls(*made)["attn"]() == -4
    rope.q_out = rope.q
    rope.ld_q = 2048                                                           # in place, rows apart
    assert calls(*made)["append"]() == -1
    cache.k_sum = None
    assert calls(*made)["select"]() == -1
    assert lib.maya_kv_read(C.byref(cache), 256, None, 3, 0, 256, 256, 256, None) == -1      # means without sums
    assert lib.maya_kv_read(C.byref(cache), 256, None, -1, 0, 256, 256, None, None) == -1
    batch.n_tokens = 0                                                         # nothing new: nothing to do
    assert all(calls(*made)[name]() == 0 for name in ("append", "attn", "select"))
    for name in ("maya_qk_norm_rope_append", "maya_block_select"):
        assert getattr(lib, name)(None, C.byref(batch), None, None) == -1


def test_rows_of_a_sequence_beyond_32_bits_are_refused(made):
    """Kernels count the rows (tokens * heads of a group) of a sequence in 32 bits."""
    lib, cache, batch, rope, attn, sel = made
    cache.n_kv = 1
    batch.n_tokens = batch.max_new = 1 << 24
    for n_q in (128, 200):
        attn.n_q, attn.ld_q = n_q, n_q * cache.head_dim
        assert calls(*made)["attn"]() == -4
