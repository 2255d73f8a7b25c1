"""What the Python handles of the attention half check and keep by themselves, on tensors of the CPU: no call gets as far as a launch."""
import pytest
import torch as T


@pytest.fixture
def api(monkeypatch):
    from project_maya_b200 import api
    monkeypatch.setattr(api, "_ptr", lambda t: None if t is None else t.data_ptr())
    return api


@pytest.fixture
def cache(api):
    return api.KvCache.empty(5, 2, 128, T.arange(4, dtype=T.int32).view(1, 4))


def test_read_refuses_outputs_of_another_size(api, cache):
    """They are written in full: one too short would be written beyond its end."""
    blocks, right = T.arange(3, dtype=T.int32), dict(k=(3, 64, 2, 128), v=(3, 64, 2, 128), mean=(3, 2, 128))
    for name, shapes in (("k", ((2, 64, 2, 128), (3, 64, 1, 128), (3, 64, 2, 64))), ("v", ((2, 64, 2, 128), (3, 32, 2, 128))),
                         ("mean", ((2, 2, 128), (3, 128), (3, 2, 64)))):
        for shape in shapes:
            out = {n: T.empty(shape if n == name else s, dtype=T.bfloat16) for n, s in right.items()}
            with pytest.raises(AssertionError):
                cache.read(blocks, **out)


def test_append_refuses_norm_weights_of_another_size(api, cache):
    """Shorter ones would be read beyond their end, longer ones be taken for their first head's."""
    batch, attn = api.AttnBatch.of([1], [3], device="cpu"), api.KvAttention(cache, 2)
    q, k, v = (T.zeros((1, 2, 128)) for _ in range(3))
    for kw in (dict(q_w=T.ones(64)), dict(k_w=T.ones(64)), dict(q_w=T.ones(256)), dict(q_w=T.ones(128), k_w=T.ones(127)), dict(q_w=T.ones((2, 128)))):
        with pytest.raises(AssertionError, match="weights"):
            attn.append(batch, q, k, v, api.Rope(**kw))


def test_attention_objects_that_share_a_rotation_keep_their_own_arguments(api, cache, monkeypatch):
    """A Rope without norms is the same for every layer; a call's pointers must not be written into it, where another thread's call would find them."""
    seen = []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def maya_qk_norm_rope_append(self, c, b, r, stream):
            seen.append((r._obj, r._obj.q, r._obj.k, r._obj.q_out, r._obj.n_q, r._obj.cos, r._obj.rot_dim))
            return 0

    real = api._lib.load()
    monkeypatch.setattr(api._lib, "load", Library)
    monkeypatch.setattr(api, "_stream", lambda stream: 0)
    monkeypatch.setattr(api, "_rows", lambda x, n, heads, dim: (x.data_ptr(), heads * dim))
    rope = api.Rope(T.ones((9, 64)), T.zeros((9, 64)))
    batch, k = api.AttnBatch.of([1], [3], device="cpu"), T.zeros((1, 2, 128))
    layers = [(api.KvAttention(cache, heads), T.zeros((1, heads, 128))) for heads in (2, 4)]
    outs = [attn.append(batch, q, k, k, rope) for attn, q in layers]
    layers[0][0].append(batch, layers[0][1], None, None, rope, q_out=outs[0])
    assert seen[0][0] is not seen[1][0] and seen[0][0] is not rope.args and seen[1][0] is not rope.args
    for (_, q_ptr, k_ptr, out, n_q, cos, rot), (attn, q), o, keys in zip(seen, [*layers, layers[0]], [*outs, outs[0]], (k, k, None)):
        assert (q_ptr, k_ptr, out, n_q) == (q.data_ptr(), None if keys is None else k.data_ptr(), o.data_ptr(), q.shape[1])
        assert cos == rope._keep[0].data_ptr() and rot == 128
    assert rope.args.q is None and rope.args.k is None and rope.args.q_out is None and rope.args.n_q == 0


def test_error_sets_the_scratch_back(api, cache, monkeypatch):
    """A launch that gave up leaves its counters somewhere in between: the next ones would start from there."""
    real, code = api._lib.load(), [1]

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def maya_attn_error(self, scratch, stream):
            return code[0]

    monkeypatch.setattr(api._lib, "load", Library)
    monkeypatch.setattr(api, "_stream", lambda stream: 0)
    attn = api.KvAttention(cache, 2)
    attn.scratch[:256] = 7
    assert attn.error() == 1 and not attn.scratch[:256].any()
    code[0] = 0
    attn.scratch[:256] = 7                                                     # (nothing wrong: nothing written)
    assert attn.error() == 0 and (attn.scratch[:256] == 7).all()
