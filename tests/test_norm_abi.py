"""Refusals of the norm with 8-bit rows on a machine without a GPU: nothing is launched, a status says why."""
import ctypes as C

import pytest
import torch as T

from project_maya_b200 import _lib, api

ARG, LIMIT = -1, -4
P = 0x7f0000000000                       # an address that nothing reads


def args(**more):
    a = _lib.RmsArgs(h=P, w=P + (1 << 20), xq=P + (2 << 20), ld_h=512, ld_add=512, ld_h_out=512, ld_x=512, n_rows=2, n=512, eps=1e-6, image=1)
    for k, v in more.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("more,status", [
    (dict(h=None), ARG), (dict(w=None), ARG), (dict(n=0), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(xq=None), ARG), (dict(xq=None, image=0), ARG), (dict(image=0), ARG),
    (dict(image=3), ARG), (dict(n=40, xq=P), ARG), (dict(xq=P + 8), ARG), (dict(n=32800, ld_h=32800), LIMIT), (dict(n_rows=1 << 31), LIMIT),
    (dict(ld_h=511), ARG), (dict(add=P, ld_add=100), ARG), (dict(h_out=P + 64, ld_h_out=500), ARG), (dict(x_out=P + 64, ld_x=500), ARG),
    (dict(h_out=P, ld_h_out=520), ARG), (dict(x_out=P, ld_x=520), ARG), (dict(x_out=P, x_is_bf16=1), ARG), (dict(x_out=P + 64, h_out=P + 64), ARG),
    (dict(add=P + 64, h_out=P + 64, add_is_bf16=1), ARG), (dict(x_out=P + (2 << 20)), ARG), (dict(add=P + 64, x_out=P + 64, ld_x=520), ARG)])
def test_refusals(lib, more, status):
    errors = lib.maya_launch_errors()
    assert lib.maya_rms_q8(C.byref(args(**more)), None) == status
    assert lib.maya_launch_errors() == errors + 1


def test_no_rows_is_no_work(lib):
    errors = lib.maya_launch_errors()
    assert lib.maya_rms_q8(C.byref(args(n_rows=0)), None) == 0
    assert lib.maya_q8_read(P, 1, 0, 64, 0, P, P, None) == 0
    assert lib.maya_launch_errors() == errors


@pytest.mark.parametrize("call", [(None, 1, 2, 64, 0, P, P), (P, 1, 2, 64, 0, None, None), (P, 0, 2, 64, 0, P, P), (P, 3, 2, 64, 0, P, P),
                                  (P, 1, 2, 48, 0, P, P), (P + 4, 1, 2, 64, 0, P, P), (P, 1, 2, 64, 0, P + 8, P), (P, 1, 2, 64, 0, P, P + 1)])
def test_read_refusals(lib, call):
    assert lib.maya_q8_read(*call, None) == ARG


def test_tensors_of_the_cpu_are_refused():
    h, w = T.zeros((2, 64)), T.ones(64)
    with pytest.raises(api.MayaError):
        api.rms_q8(h, None, w, 1e-6)
    with pytest.raises(api.MayaError):
        api.q8_read(T.zeros(144, dtype=T.uint8), 2, 64)


def test_sizes():
    assert api.xq_bytes(api.XQ_Q8_1, 3, 64) == 3 * 72
    assert api.xq_bytes(api.XQ_MMQ, 3, 64) == 3 * 2 * (64 + 64)
