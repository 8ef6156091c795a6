"""What the 8-bit kept form refuses, before anything is launched."""

import pytest
import torch

from mlops_b200 import layer, ops, provider
from mlops_b200._lib import NativeError, lib


def test_cpu_tensors_are_refused():
    h = torch.zeros(4, 256, dtype=torch.bfloat16)
    saved = (torch.zeros(4, 256, dtype=torch.int8), torch.zeros(4, 2))
    for call in (lambda: ops.swiglu_save8(h), lambda: ops.restore8(saved),
                 lambda: ops.dswiglu_saved8(saved, h[:, :128], torch.zeros(4), torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(NativeError, match="CUDA"):
            call()


def test_layouts_other_than_the_kept_one_are_refused():
    codes, scales = torch.zeros(4, 256, dtype=torch.int8), torch.zeros(4, 2)
    assert ops._check_saved(codes, scales) == (4, 128)
    assert ops._check_saved(torch.zeros(0, 272, dtype=torch.int8), torch.zeros(0, 4)) == (0, 136)
    for bad in ((codes.to(torch.uint8), scales), (codes[:, :250], scales), (codes.t().contiguous().t(), scales),
                (codes, scales.double()), (codes, torch.zeros(4, 4)), (codes, torch.zeros(3, 2)), (codes[0], scales)):
        with pytest.raises(NativeError):
            ops._check_saved(*bad)


def test_the_entry_points_refuse_bad_pointers_and_pitches():
    """Invented addresses: every call ends before its launch."""
    p = 4096
    save = lambda h=p, ldh=256, rows=4, width=128, codes=p, ld=256, scales=p: lib.b200moe_swiglu_save8(  # noqa: E731
        h, ldh, rows, width, None, 128, None, 0, 0, None, 128, codes, ld, scales, 2, 1, 0.0, 0, None)
    assert save(h=None) == -1 and save(codes=None) == -1 and save(scales=None) == -1 and save(rows=-1) == -1
    assert save(width=0) == -1 and save(width=100) == -2 and save(ld=250) == -2 and save(codes=p + 4) == -2
    assert save(h=p + 8) == -2 and save(ldh=252) == -2 and save(rows=0) == 0
    restore = lambda codes=p, out=p, width=128, ldo=256: lib.b200moe_restore8(  # noqa: E731
        codes, 256, p, 2, 1, 4, width, out, ldo, None)
    assert restore(codes=None) == -1 and restore(out=None) == -1 and restore(width=4) == -2 and restore(ldo=4) == -2
    back = lambda codes=p, r=p, weights=p, n=4, order=p, q=None, qs=None, status=p: lib.b200moe_dswiglu_saved8(  # noqa: E731
        codes, 256, p, 2, 1, r, 128, weights, n, order, 4, 128, p, q, 256, qs, 1, 4, None, 256, None, 128, 0.0, 0,
        status, None)
    assert back(codes=None) == -1 and back(r=None) == -1 and back(weights=None) == -1 and back(n=0) == -1
    assert back(order=None) == -1 and back(q=p) == -1 and back(status=None) == -1 and back(r=p + 8) == -2


def test_the_one_call_layer_refuses_a_missing_kept_form():
    import ctypes

    from mlops_b200._lib import BackwardArgs, ForwardArgs

    sizes = dict(tokens=4, width=256, inner=128, experts=8, top_k=2)

    def filled(struct, **changes):
        pointers = [name for name, kind in struct._fields_ if kind is ctypes.c_void_p]
        return ctypes.byref(struct(**{**sizes, "mode": 1, **{name: 4096 for name in pointers}, **changes}))

    assert lib.b200moe_forward_fp8_save8(filled(ForwardArgs), None, 4096, None) == -1
    assert lib.b200moe_forward_fp8_save8(filled(ForwardArgs), 4096, None, None) == -1
    assert lib.b200moe_forward_fp8_save8(filled(ForwardArgs), 4096 + 8, 4096, None) == -2
    assert lib.b200moe_forward_fp8_save8(None, 4096, 4096, None) == -1
    assert lib.b200moe_backward_fp8_saved8(filled(BackwardArgs, h13=None), None, 4096, None) == -1
    assert lib.b200moe_backward_fp8_saved8(filled(BackwardArgs, h13=None), 4096, None, None) == -1
    assert lib.b200moe_backward_fp8_saved8(filled(BackwardArgs, h13=None), 4096 + 8, 4096, None) == -2


def test_the_setting_takes_the_two_forms_only():
    assert provider.set_saved_activations("int8") == "bf16"
    assert provider.set_saved_activations("bf16") == "int8"
    with pytest.raises(ValueError):
        provider.set_saved_activations("fp8")
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="saved"):
        layer.forward_routed(x, x, None, None, None, top_k=1, routing_mode="softmax_then_topk", saved="int4")
    with pytest.raises(ValueError, match="fuse_swiglu"):
        layer.forward_routed(x, x, None, None, None, top_k=1, routing_mode="softmax_then_topk", saved="int8",
                             fuse_swiglu=True)
