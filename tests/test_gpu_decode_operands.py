"""Operands of the layer for a few tokens that `forward_routed` and `provider.apply` take and its kernels do not read as they
are: they are converted, or the call says what it does not take."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(T=5, D=256, F=128, E=8):
    g = torch.Generator().manual_seed(7)
    new = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16().to(DEV)  # noqa: E731
    return new(T, D), new(T, D), new(E, D, std=0.1), new(E, 2 * F, D, std=0.1), new(E, D, F, std=0.1)


def _off(t, elements=1):
    """The same values in a piece of a larger buffer that starts at an odd address."""
    flat = torch.empty(t.numel() + elements, dtype=t.dtype, device=t.device)
    flat[elements:] = t.reshape(-1)
    return flat[elements:].view(t.shape)


@pytest.mark.parametrize("kind", ["float16", "float64", "strided", "transposed", "odd address", "odd address, fp32"])
def test_routers_of_other_types_strides_and_addresses(kind):
    from mlops_b200 import layer

    x, residual, router, w13, w2 = _inputs()
    call = lambda r: layer.forward_decode(x, residual, r, w13, w2, top_k=2, routing_mode="softmax_then_topk")  # noqa: E731
    router = router.to(torch.float16).to(torch.bfloat16)  # values that every type holds
    wide = torch.zeros(8, 512, dtype=torch.bfloat16, device=DEV)
    wide[:, :256] = router
    other = {"float16": router.half(), "float64": router.double(), "strided": wide[:, :256],
             "transposed": router.t().contiguous().t(), "odd address": _off(router),
             "odd address, fp32": _off(router.float())}[kind]
    assert all(torch.equal(a, b) for a, b in zip(call(other), call(router)))


def test_shared_weights_at_odd_addresses():
    """They take the library products of `apply`, as strided ones do."""
    from mlops_b200 import provider

    x, residual, router, w13, w2 = _inputs()
    g = torch.Generator().manual_seed(8)
    shared = [(torch.randn(*shape, generator=g) * 0.1).bfloat16().to(DEV) for shape in ((128, 256), (256, 64))]
    call = lambda residual, **kw: provider.decode(x, residual, router, w13, w2, top_k=2,  # noqa: E731
                                                  routing_mode="softmax_then_topk", swiglu_limit=1, **kw)
    expected = call(residual + provider.shared_expert(x, *shared, swiglu_limit=1.0))
    for one, other in ((_off(shared[0]), shared[1]), (shared[0], _off(shared[1], 3))):
        assert torch.equal(call(residual, shared_w13=one, shared_w2=other), expected)


def test_sizes_past_the_limit_are_named():
    from mlops_b200 import layer, ops

    x = torch.zeros(1, 2 ** 19 + 8, dtype=torch.bfloat16, device=DEV)
    router = torch.zeros(1, x.shape[1], dtype=torch.bfloat16, device=DEV)
    w13 = torch.zeros(1, 16, x.shape[1], dtype=torch.bfloat16, device=DEV)
    w2 = torch.zeros(1, x.shape[1], 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ops.NativeError, match="at most"):
        layer.forward_decode(x, x, router, w13, w2, top_k=1, routing_mode="softmax_then_topk")
