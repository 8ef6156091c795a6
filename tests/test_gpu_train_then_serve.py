"""The kept 8-bit form and the layer for a few tokens as a program uses them together: steps of training with int8
activations on fp32 masters, publication into the block-FP8 containers, decoding from them."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_train_publish_decode():
    from mlops_b200 import layer, ops, provider
    from mlops_b200.weights import BlockFP8Weight

    g = torch.Generator().manual_seed(0)
    rand = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).to(DEV)  # noqa: E731
    D, F, E, K, T = 256, 128, 8, 2, 192
    masters = [rand(E, 2 * F, D, std=0.08), rand(E, D, F, std=0.08)]
    router = rand(E, D, std=0.1).requires_grad_(True)
    shared = [rand(2 * F, D, std=0.06).bfloat16().requires_grad_(True), rand(D, F, std=0.08).bfloat16().requires_grad_(True)]
    containers = [BlockFP8Weight.quantize(m) for m in masters]
    for c in containers:
        c.requires_grad_(True)
    routing = dict(top_k=K, routing_mode="softmax_then_topk")
    x, residual, dy = (rand(T, D).bfloat16() for _ in range(3))
    prompt = x[:4].clone()
    previous = provider.set_saved_activations("int8")
    try:
        for _ in range(3):
            out, *_ = provider.apply(x, residual, router, *containers, shared_w13=shared[0], shared_w2=shared[1], **routing)
            grads = torch.autograd.grad(out, [router, *containers, *shared], dy)
            assert all(bool(t.isfinite().all()) for t in grads)
            with torch.no_grad():
                for t, step in zip((router, *shared), (grads[0], *grads[3:])):
                    t -= 1e-3 * step.to(t.dtype)
                for master, container, step in zip(masters, containers, grads[1:3]):
                    before = container._data.clone()
                    master -= 1e-3 * step.float()
                    container.copy_(master)
                    assert not torch.equal(before.view(torch.uint8), container._data.view(torch.uint8))
    finally:
        provider.set_saved_activations(previous)

    extra = dict(shared_w13=shared[0], shared_w2=shared[1])
    with torch.no_grad():
        served = provider.decode(prompt, residual[:4], router, *containers, **extra, **routing)
        raw, weights, ids = layer.forward_decode(
            prompt, residual[:4], router, *((c._data, c._scale) for c in containers), shared=tuple(shared), **routing)
        full, *_ = provider.apply(prompt, residual[:4], router, *containers, **extra, **routing)
    assert torch.equal(served, raw)
    ops.check_status(DEV)

    # the decoded output from the published weights in 64 bits (tolerance: tests/test_gpu_decode.py)
    values = [(c._data.double() * c._scale.double().repeat_interleave(128, 1).repeat_interleave(128, 2)).cpu()
              for c in containers]
    xs, expected = prompt.double().cpu(), residual[:4].double().cpu()
    size = torch.zeros_like(expected)
    terms = [(values[0][e], values[1][e], (weights * (ids == e)).sum(1).double().cpu()) for e in range(E)]
    terms.append((shared[0].detach().double().cpu(), shared[1].detach().double().cpu(), torch.ones(4).double()))
    for w13, w2, share in terms:
        gate, up = (xs @ w13.t()).chunk(2, -1)
        act = (gate * torch.sigmoid(gate) * up).bfloat16().double() * share[:, None]
        expected += act @ w2.t()
        size += act.abs() @ w2.abs().t()
    tolerance = 2.0 ** -8 * expected.abs() + (0.02 * 2.0 ** -7 + 500 * 2.0 ** -24 + 4e-5) * size
    assert bool(((served.double().cpu() - expected).abs() <= tolerance).all())
    # and near the training layer's own output: its activations carry two E4M3 roundings, 2.6% rms each
    assert float((full.float() - served.float()).norm() / served.float().norm()) < 0.06


def test_decode_takes_what_apply_takes():
    from mlops_b200 import provider
    from mlops_b200.weights import BlockFP8Weight

    g = torch.Generator().manual_seed(1)
    rand = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16().to(DEV)  # noqa: E731
    x, residual, router = rand(3, 256), rand(3, 256), rand(8, 256, std=0.1).float()
    w13, w2 = rand(8, 256, 256, std=0.08), rand(8, 256, 128, std=0.08)
    routing = dict(top_k=2, routing_mode="sigmoid_noaux_tc", router_bias=torch.randn(8, device=DEV) * 0.1, n_group=4,
                   topk_group=2, routed_scaling=2.5, swiglu_limit=2.0)
    odd = dict(shared_w13=rand(200, 256, std=0.06), shared_w2=rand(256, 100, std=0.08))
    for call in (provider.apply, provider.decode):  # an activation pitch that is not a multiple of 16 bytes: neither
        with torch.no_grad(), pytest.raises(Exception):
            call(x, residual, router, w13, w2, **routing, **odd)
    shared = dict(shared_w13=rand(208, 256, std=0.06), shared_w2=rand(256, 104, std=0.08))
    columns = dict(shared_w13=rand(256, 208, std=0.06).t(), shared_w2=shared["shared_w2"])  # strides of a transpose
    gate = rand(1, 256, std=0.1)
    for weights in ((w13, w2), (BlockFP8Weight.quantize(w13), BlockFP8Weight.quantize(w2))):
        for extra in ({}, shared, columns, dict(shared_w13=shared["shared_w13"], shared_w2=shared["shared_w2"],
                                       shared_gate_weight=gate, shared_mode="sigmoid")):
            with torch.no_grad():
                full = provider.apply(x, residual, router, *weights, **routing, **extra)[0]
                few = provider.decode(x, residual, router, *weights, **routing, **extra)
            assert float((full.float() - few.float()).norm() / few.float().norm()) < 0.06
    x.requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        provider.decode(x, residual, router, w13, w2, **routing)
    many = torch.zeros(65, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="64 tokens"):
        provider.decode(many, many, router, w13, w2, **routing)
