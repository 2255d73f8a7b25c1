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
    for name, shapes in (("k", ((2, 64, 2, 128), (3, 64, 1, 128), (3, 64, 2, 64), (3 * 64 * 2 * 128,))), ("v", ((2, 64, 2, 128), (3, 32, 2, 128))),
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
