"""`provider.decode` where tensors are traced or counted instead of run: it is one registered operator there."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T, D, F, E, K, FS = 5, 256, 128, 8, 2, 64


def _inputs(fp8):
    from mlops_b200.weights import BlockFP8Weight

    g = torch.Generator().manual_seed(7)
    new = lambda *shape, std=0.1: (torch.randn(*shape, generator=g) * std).bfloat16().to(DEV)  # noqa: E731
    w13, w2 = new(E, 2 * F, D), new(E, D, F)
    if fp8:
        w13, w2 = BlockFP8Weight.quantize(w13), BlockFP8Weight.quantize(w2)
    shared = dict(shared_w13=new(2 * FS, D), shared_w2=new(D, FS))
    return (new(T, D, std=1.0), new(T, D, std=1.0), new(E, D), w13, w2), shared, new(1, D)


def _decode(*args, **shared):
    from mlops_b200 import provider

    return provider.decode(*args, top_k=K, routing_mode="softmax_then_topk", swiglu_limit=2.0, **shared)


def _kinds(shared, gate):
    return [{}, shared, dict(shared, shared_gate_weight=gate, shared_mode="sigmoid")]


@pytest.mark.parametrize("fp8", [False, True])
def test_one_graph_of_a_compiled_step(fp8):
    """`torch.compile` without a graph break: the same bits."""
    args, shared, gate = _inputs(fp8)
    with torch.no_grad():
        for kwargs in _kinds(shared, gate):
            expected = _decode(*args, **kwargs)
            torch._dynamo.reset()
            step = torch.compile(lambda h, **kw: _decode(h, *args[1:], **kw) * 2, fullgraph=True, backend="aot_eager")
            assert torch.equal(step(args[0], **kwargs), expected * 2)


def test_fake_tensors_pass():
    from torch._subclasses.fake_tensor import FakeTensorMode

    args, shared, gate = _inputs(False)
    with FakeTensorMode() as mode:
        fake = [mode.from_tensor(t) for t in args]
        for kwargs in _kinds({k: mode.from_tensor(v) for k, v in shared.items()}, mode.from_tensor(gate)):
            out = _decode(*fake, **kwargs)
            assert out.shape == (T, D) and out.dtype == torch.bfloat16 and out.device.type == "cuda"
            assert _decode(fake[0].view(1, T, D), fake[1].view(1, T, D), *fake[2:], **kwargs).shape == (1, T, D)


@pytest.mark.parametrize("fp8", [False, True])
def test_the_products_are_counted(fp8):
    from torch.utils.flop_counter import FlopCounterMode

    args, shared, gate = _inputs(fp8)
    from mlops_b200 import provider

    routed = provider._logical_flops(*args[:1], *args[2:], K, True)
    for kwargs in _kinds(shared, gate):
        with FlopCounterMode(display=False) as count:
            out = _decode(*args, **kwargs)
        assert count.get_total_flops() == routed + (T * (6 * D * FS + 5 * FS) if kwargs else 0)
        assert torch.equal(out, _decode(*args, **kwargs))


def test_the_operator_keeps_the_contract():
    from mlops_b200 import provider

    args, shared, gate = _inputs(False)
    none = torch.empty(0, device=DEV)
    torch.library.opcheck(provider.moe_decode, (*args, none, K, "softmax_then_topk", 1, 1, 1.0, None, "add",
                                                list(shared.values()), []), test_utils=("test_schema", "test_faketensor"))


def test_a_forward_mode_tangent_is_refused():
    import torch.autograd.forward_ad as forward_ad

    args, shared, gate = _inputs(False)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(ValueError, match="no gradient"):
            _decode(dual, *args[1:])
        assert _decode(*args).shape == (T, D)  # a level alone changes nothing
