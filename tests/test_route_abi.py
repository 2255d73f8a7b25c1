"""Refusals of the router over groups and of the layer for routed tokens on a machine without a GPU."""
import ctypes as C

import pytest
import torch as T

from project_maya_b200 import _lib, api

ARG, LIMIT = -1, -4
P = 0x7f0000000000                       # an address that nothing reads


@pytest.mark.parametrize("more,status", [
    (dict(logits=None), ARG), (dict(ids=None), ARG), (dict(weights=None), ARG), (dict(n_expert=0), ARG), (dict(k=0), ARG), (dict(n_group=0), ARG),
    (dict(n_keep=0), ARG), (dict(n_keep=9), ARG), (dict(n_group=7), ARG), (dict(k=65, n_keep=8), LIMIT), (dict(n_expert=4096), LIMIT),
    (dict(n_group=64, n_keep=64), LIMIT), (dict(k=33, n_keep=1), LIMIT)])
def test_refusals(lib, more, status):
    a = dict(logits=P, bias=None, n_tokens=3, n_expert=256, k=8, n_group=8, n_keep=4, sigmoid=1, top2=1, norm_w=1, w_scale=1.0, ids=P, weights=P)
    errors = lib.maya_launch_errors()
    assert lib.maya_router_groups(C.byref(_lib.RouteArgs(**{**a, **more})), None) == status
    assert lib.maya_launch_errors() == errors + 1
    assert lib.maya_router_groups(C.byref(_lib.RouteArgs(**{**a, "n_tokens": 0})), None) == 0


def test_tensors_of_the_cpu_are_refused():
    with pytest.raises(api.MayaError):
        api.router_groups(T.zeros((2, 64)), 4)


def test_routed_layer_refusals(lib):
    rb = lib.maya_row_bytes
    L = _lib.MoeLayerDesc(512, 256, 32, 4, api.Q4_K, api.Q8_0, P, 2 * 256 * rb(api.Q4_K, 512) + 512 * rb(api.Q8_0, 256))
    L.limit, L.expert_hi, L.router_w_scale = float("inf"), 32, 1.0
    call = lambda **m: lib.maya_moe_layer_decode_routed(*{**dict(L=C.byref(L), ids=P, w=P, x=P, bf16=0, T=2, out=P, scratch=P, n=1 << 30, s=None), **m}.values())   # noqa: E731
    assert call(ids=None) == ARG and call(w=None) == ARG and call(x=None) == ARG and call(out=None) == ARG and call(L=None) == ARG
    assert call(T=0) == LIMIT and call(T=17) == LIMIT and call(n=64) == LIMIT and call(scratch=P + 16) == ARG
    L.n_ff_sh, L.shared, L.shared_here, L.sh_gu_type, L.sh_d_type, L.sh_lo, L.sh_hi = 256, P, 1, api.Q8_0, api.Q8_0, 0, 64
    assert call() == ARG
