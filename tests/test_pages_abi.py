"""Refusals of the cache's pages on a machine without a GPU: nothing is launched, a status says why."""
import ctypes as C

import pytest
import torch as T

from project_maya_b200 import _lib, api

ARG, LIMIT = -1, -4
P = 0x7f0000000000                       # an address that nothing reads


def desc(**more):
    d = dict(layers=P, table=P, refs=P, scratch=P, scratch_bytes=1 << 40, n_seq=4, table_ld=8, n_blocks=64, n_layers=2, n_kv=8, head_dim=128, has_sums=1)
    return C.byref(_lib.KvPagesDesc(**{**d, **more}))


def batch(**more):
    b = dict(start=P, kv_len=P, n_seq=4, n_tokens=4, max_new=1, max_len=512)
    return C.byref(_lib.AttnBatchDesc(**{**b, **more}))


@pytest.mark.parametrize("more,status", [
    (dict(layers=None), ARG), (dict(table=None), ARG), (dict(refs=None), ARG), (dict(scratch=None), ARG), (dict(scratch=P + 16), ARG), (dict(scratch_bytes=64), LIMIT),
    (dict(refs=P + 4), ARG), (dict(layers=P + 8), ARG), (dict(n_seq=0), ARG), (dict(table_ld=0), ARG), (dict(n_blocks=0), ARG), (dict(n_layers=0), ARG),
    (dict(n_kv=0), ARG), (dict(head_dim=96), LIMIT), (dict(n_blocks=(1 << 20) + 1), LIMIT), (dict(n_seq=65536), LIMIT), (dict(n_layers=1025), LIMIT),
    (dict(n_seq=60000, table_ld=8192), LIMIT)])
def test_descriptors_that_are_refused(lib, more, status):
    d = desc(**more)
    assert lib.maya_pages_reserve(d, batch(), None) == status
    assert lib.maya_pages_fork(d, P, P, P, 2, None) == status
    assert lib.maya_pages_free(d, P, 2, None) == status
    assert lib.maya_pages_compact(d, 64, None) == status
    assert lib.maya_pages_copy(d, P, P, 2, None) == status
    if not {"scratch", "scratch_bytes", "refs", "layers"} & set(more):
        assert lib.maya_pages_scratch_bytes(d) == 0
    assert lib.maya_pages_reserve(None, batch(), None) == ARG and lib.maya_pages_scratch_bytes(None) == 0


def test_calls_that_are_refused(lib):
    d = desc()
    assert lib.maya_pages_scratch_bytes(d) >= 4 * (3 * 64 + 2 * 4 + 32)
    for more in (dict(start=None), dict(kv_len=None), dict(n_seq=5), dict(n_seq=-1), dict(n_tokens=-1), dict(max_new=0), dict(max_len=513), dict(n_seq=0)):
        assert lib.maya_pages_reserve(d, batch(**more), None) == ARG, more
    assert lib.maya_pages_reserve(d, batch(n_tokens=(1 << 24) + 1), None) == LIMIT
    assert lib.maya_pages_reserve(d, None, None) == ARG
    assert lib.maya_pages_fork(d, None, P, P, 2, None) == ARG and lib.maya_pages_fork(d, P, P, P, -1, None) == ARG
    assert lib.maya_pages_fork(d, P, P, P, 5, None) == LIMIT
    assert lib.maya_pages_free(d, None, 1, None) == ARG and lib.maya_pages_free(d, P, -1, None) == ARG
    assert lib.maya_pages_copy(d, P, None, 1, None) == ARG and lib.maya_pages_copy(d, P, P, 65, None) == LIMIT
    assert lib.maya_pages_error(None, None) == ARG and lib.maya_pages_compact(d, -1, None) == ARG


def test_nothing_to_do_is_no_launch(lib):
    d, n = desc(), lib.maya_launch_count()
    assert lib.maya_pages_reserve(d, batch(n_tokens=0), None) == 0 and lib.maya_pages_reserve(d, batch(max_len=0), None) == 0
    assert lib.maya_pages_fork(d, P, P, P, 0, None) == 0 and lib.maya_pages_free(d, P, 0, None) == 0 and lib.maya_pages_copy(d, P, P, 0, None) == 0
    assert lib.maya_launch_count() == n


def test_caches_of_other_tables_or_shapes_are_refused(monkeypatch):
    monkeypatch.setattr(api, "_ptr", lambda t: None if t is None else t.data_ptr())
    table = T.full((2, 4), -1, dtype=T.int32)
    a = api.KvCache.empty(8, 2, 64, table)
    for b in (api.KvCache.empty(8, 2, 64, table.clone()), api.KvCache.empty(9, 2, 64, table), api.KvCache.empty(8, 1, 64, table),
              api.KvCache.empty(8, 2, 128, table), api.KvCache.empty(8, 2, 64, table, sums=False)):
        with pytest.raises(AssertionError):
            api.KvPages([a, b])
    pages = api.KvPages([a, api.KvCache.empty(8, 2, 64, table)])
    assert pages.refs.tolist() == [0] * 8
    with pytest.raises(api.MayaError):                       # tensors of the CPU
        pages.compact()
    with pytest.raises(AssertionError):
        api.KvPages([a], refs=T.zeros(7, dtype=T.int32))


def test_rows_of_more_tokens_than_an_int_counts_are_refused(lib):
    """64 * table_ld is a number of tokens: at 2^25 blocks a row it would wrap, and a fork would leave the children nothing."""
    assert lib.maya_pages_scratch_bytes(desc(n_seq=1, table_ld=(1 << 25) - 1)) > 0
    for wide in (1 << 25, 1 << 26):
        d = desc(n_seq=1, table_ld=wide)
        assert lib.maya_pages_scratch_bytes(d) == 0
        assert lib.maya_pages_fork(d, P, P, P, 1, None) == LIMIT and lib.maya_pages_reserve(d, batch(n_seq=1), None) == LIMIT
        assert lib.maya_pages_free(d, P, 1, None) == LIMIT and lib.maya_pages_compact(d, 1, None) == LIMIT and lib.maya_pages_copy(d, P, P, 1, None) == LIMIT


def test_caches_in_parts_on_two_devices_are_refused(monkeypatch):
    """A cache's buffers go to the kernels by address: they all have to lie where the table does."""
    monkeypatch.setattr(api, "_ptr", lambda t: None if t is None else t.data_ptr())
    table = T.full((2, 4), -1, dtype=T.int32)
    c = api.KvCache.empty(8, 2, 64, table)
    parts = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale, table=table, k_sum=c.k_sum)
    assert api.KvPages([api.KvCache(**parts)]).n_blocks == 8
    for name in parts:
        with pytest.raises(AssertionError):
            api.KvPages([api.KvCache(**{**parts, name: parts[name].to("meta")})], refs=T.zeros(8, dtype=T.int32))
