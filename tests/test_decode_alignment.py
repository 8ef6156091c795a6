"""Addresses that the layer for a few tokens and the layer with a kept form in 8 bits refuse: invented ones, every call
ends before its first launch."""

import ctypes

import pytest

from mlops_b200._lib import BackwardArgs, DecodeArgs, ForwardArgs, lib


def _filled(struct, sizes, **changes):
    pointers = [name for name, kind in struct._fields_ if kind is ctypes.c_void_p]
    return ctypes.byref(struct(**{**sizes, **{name: 4096 for name in pointers}, **changes}))


@pytest.mark.parametrize("name", ["w13_scale", "w2_scale", "bias", "route_weights", "ids", "status"])
def test_words_at_odd_addresses_are_refused(name):
    sizes = dict(tokens=4, width=256, inner=128, experts=8, top_k=2, mode=1, n_group=1, topk_group=1)
    assert lib.b200moe_decode(_filled(DecodeArgs, sizes, **{name: 4096 + 2}), None) == -2


def test_the_one_call_layer_refuses_code_scales_at_an_odd_address_before_it_launches():
    sizes = dict(tokens=4, width=256, inner=128, experts=8, top_k=2, mode=1)
    assert lib.b200moe_forward_fp8_save8(_filled(ForwardArgs, sizes), 4096, 4096 + 2, None) == -2
    assert lib.b200moe_backward_fp8_saved8(_filled(BackwardArgs, sizes, h13=None), 4096, 4096 + 2, None) == -2
