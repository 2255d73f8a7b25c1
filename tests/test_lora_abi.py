"""Refusals of the low-rank adapters on a machine without a GPU: nothing is launched, a status says why."""
import ctypes as C

import pytest
import torch as T

from project_maya_b200 import _lib, api

ARG, LIMIT = -1, -4
P = 0x7f0000000000                       # an address that nothing reads


@pytest.mark.parametrize("more,status", [
    (dict(x=None), ARG), (dict(out=None), ARG), (dict(a=None), ARG), (dict(b=None), ARG), (dict(idx=None), ARG), (dict(scratch=None), ARG),
    (dict(n_adapters=0), ARG), (dict(n_in=0), ARG), (dict(n_in=48, ld_x=64), ARG), (dict(n_out=0), ARG), (dict(rank=0), ARG), (dict(rank=8), ARG), (dict(rank=272), LIMIT),
    (dict(n_tokens=65536), LIMIT), (dict(ld_x=32), ARG), (dict(ld_y=32), ARG), (dict(ld_out=32), ARG), (dict(y=P, out=P, ld_out=128), ARG), (dict(x=P + 4), ARG),
    (dict(a=P + 8), ARG), (dict(b=P + 8), ARG), (dict(scratch=P + 128), ARG), (dict(ld_x=66), ARG), (dict(ld_x=68, x_is_bf16=1), ARG), (dict(scratch_bytes=100), LIMIT), (dict(ld_out=1 << 31), LIMIT), (dict(kernel=3), ARG), (dict(kernel=-1), ARG),
    (dict(kernel=2, n_adapters=4097), LIMIT), (dict(kernel=2, scratch_bytes=1000), LIMIT)])
def test_refusals(lib, more, status):
    d = dict(x=P, y=P + 4096, out=P + 8192, a=P, b=P, scale=None, idx=P, scratch=P, scratch_bytes=1 << 30, ld_x=64, ld_y=64, ld_out=64, n_tokens=3, n_in=64, n_out=64,
             rank=16, n_adapters=2, x_is_bf16=0, w_is_f16=0)
    errors = lib.maya_launch_errors()
    assert lib.maya_lora(C.byref(_lib.LoraArgs(**{**d, **more})), None) == status
    assert lib.maya_launch_errors() == errors + 1
    assert lib.maya_lora(C.byref(_lib.LoraArgs(**{**d, "n_tokens": 0})), None) == 0


def test_scratch_sizes(lib):
    f = lib.maya_lora_scratch_bytes
    assert f(64, 16, 2, 100) > 0 and f(4096, 256, 1000, 65535) > 0
    for bad in ((0, 16, 2, 1), (48, 16, 2, 1), (64, 8, 2, 1), (64, 272, 2, 1), (64, 16, 0, 1), (64, 16, 2, 0), (64, 16, 2, 65536)):
        assert f(*bad) == 0
    for small, large in ((1, 2), (100, 129), (1000, 4096)):                    # more tokens never need less
        assert f(512, 32, 4, small) <= f(512, 32, 4, large)


def test_adapters_of_other_shapes_or_types_are_refused(monkeypatch):
    monkeypatch.setattr(api, "_ptr", lambda t: None if t is None else t.data_ptr())
    a, b = T.zeros((2, 16, 64)).half(), T.zeros((2, 96, 16)).half()
    ad = api.LoraAdapters(a, b, T.ones(2))
    assert (ad.rank, ad.n_in, ad.n_out) == (16, 64, 96)
    padded = api.LoraAdapters(a[:, :5], b[..., :5])
    assert padded.rank == 16 and padded.a.shape == a.shape and padded.b.shape == b.shape
    for args in ((a, b.bfloat16()), (a.float(), b.float()), (a, b[:1]), (a, b[..., :8]), (a, b, T.ones(3)), (a, b, T.ones(2).half())):
        with pytest.raises(AssertionError):
            api.LoraAdapters(*args)
    with pytest.raises(api.MayaError):
        api.LoraAdapters(a[..., :40].contiguous(), b)
    with pytest.raises(api.MayaError):                       # tensors of the CPU
        ad.forward(T.zeros((1, 64)), T.zeros(1, dtype=T.int32))


def test_adapters_on_two_devices_are_refused(monkeypatch):
    """b and scale go to the kernels by address: they have to lie where a does."""
    monkeypatch.setattr(api, "_ptr", lambda t: None if t is None else t.data_ptr())
    a, b = T.zeros((2, 16, 64)).half(), T.zeros((2, 96, 16)).half()
    for args in ((a, b.to("meta")), (a, b, T.ones(2, device="meta"))):
        with pytest.raises(AssertionError):
            api.LoraAdapters(*args)
