"""What the layer for a few tokens refuses, before anything is launched."""

import ctypes

import pytest
import torch

from mlops_b200 import layer, ops
from mlops_b200._lib import DecodeArgs, NativeError, lib

SIZES = dict(tokens=4, width=256, inner=128, experts=8, top_k=2, mode=1, n_group=1, topk_group=1)
OPTIONAL = {"bias", "shared_w13", "shared_w2"}


def _filled(**changes):
    pointers = [name for name, kind in DecodeArgs._fields_ if kind is ctypes.c_void_p]
    return ctypes.byref(DecodeArgs(**{**SIZES, **{name: 4096 for name in pointers}, **changes}))


def test_the_argument_struct_is_laid_out_like_the_headers():
    import re
    from pathlib import Path

    header = Path(__file__).resolve().parent.parent / "include" / "b200moe.h"
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    body = re.search(r"typedef struct b200moe_decode_args \{(.*?)\}", text, flags=re.S).group(1)
    kinds = {"long long": ctypes.c_longlong, "int": ctypes.c_int, "float": ctypes.c_float}
    declared = []
    for line in filter(str.strip, body.split(";")):
        if "*" in line:
            declared.append((line.split("*")[1].strip(), ctypes.c_void_p))
        else:
            kind = next(k for k in kinds if line.strip().startswith(k))
            declared += [(n.strip(), kinds[kind]) for n in line.strip()[len(kind):].split(",")]
    assert declared == list(DecodeArgs._fields_)


def test_the_entry_point_refuses_bad_arguments_before_any_launch():
    """Invented addresses: every call ends before its first launch."""
    call = lambda **changes: lib.b200moe_decode(_filled(**changes), None)  # noqa: E731
    assert lib.b200moe_decode(None, None) == -1
    for name, kind in DecodeArgs._fields_:
        if kind is ctypes.c_void_p and name not in OPTIONAL:
            assert call(**{name: None}) == -1, name
    assert call(shared_inner=128, shared_w13=None) == -1 and call(shared_inner=128, shared_w2=None) == -1
    assert call(tokens=-1) == -1 and call(tokens=65) == -6 and call(experts=1025) == -6 and call(top_k=9) == -1
    assert call(top_k=0) == -1 and call(experts=64, top_k=33) == -6 and call(mode=3) == -1 and call(mode=-1) == -1
    assert call(width=200) == -2 and call(inner=100) == -2 and call(shared_inner=12) == -2
    assert call(width=204, w13_scale=None, w2_scale=None) == -2
    assert call(mode=2, n_group=3) == -1 and call(mode=2, n_group=0) == -1 and call(mode=2, topk_group=0) == -1
    assert call(experts=64, mode=2, n_group=64, topk_group=2) == -6
    for name in ("x", "router", "w13", "w2"):
        assert call(**{name: 4096 + 8}) == -2, name
    assert call(workspace=4096 + 128) == -2 and call(tokens=0) == 0
    assert lib.b200moe_decode_workspace_bytes(65, 256, 128, 8, 2, 0) == -1
    with_shared = [lib.b200moe_decode_workspace_bytes(4, 256, 128, 8, 2, shared) for shared in (0, 128)]
    assert with_shared[1] - with_shared[0] == 2 * 4 * 128 + 4 * 4 * 256  # its activation and its rows of y


def test_the_wrapper_refuses_what_it_does_not_take():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    router = torch.zeros(8, 256)
    w13, w2 = torch.zeros(8, 256, 256, dtype=torch.bfloat16), torch.zeros(8, 256, 128, dtype=torch.bfloat16)
    fp8 = lambda w: (w.to(torch.float8_e4m3fn), torch.ones(w.shape[0], w.shape[1] // 128, w.shape[2] // 128))  # noqa: E731
    call = lambda w13=w13, w2=w2, **kw: layer.forward_decode(  # noqa: E731
        x, x, router, w13, w2, **{**dict(top_k=2, routing_mode="softmax_then_topk"), **kw})
    for first, second in ((w13, w2), (fp8(w13), fp8(w2))):  # CPU tensors
        with pytest.raises(NativeError, match="CUDA"):
            call(first, second)
    for first, second in ((fp8(w13), w2), (w13, fp8(w2)), (w13.float(), w2.float()), (w13[:4], w2),
                          (w13.transpose(1, 2), w2), (fp8(w13)[:1] + (torch.ones(8, 2, 1),), fp8(w2)),
                          ((fp8(w13)[0], fp8(w13)[1].double()), fp8(w2)), (w13[0], w2[0])):
        with pytest.raises(NativeError):
            call(first, second)
    assert ops.DECODE_TOKENS == 64


def test_the_provider_refuses_with_the_reason():
    from mlops_b200 import provider

    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    w13, w2 = torch.zeros(8, 256, 256, dtype=torch.bfloat16), torch.zeros(8, 256, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        provider.decode(x, x, torch.zeros(8, 256), w13, w2, top_k=2, routing_mode="softmax_then_topk")
