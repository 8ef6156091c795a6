"""The layer for a few tokens at wide experts: 28 blocks of output columns, 112 K blocks of the down product, rows of act
that a block of 1024 threads scales. Against the formula in 64 bits on the GPU.

Tolerance of an output: its own rounding to bf16, 2^-8 of it; the activation's rounding is in the formula, and the fp32
sums before it (relative error about sqrt(D) 2^-24 of sum|x w|) let under 1% of them round the other way: twice that,
0.02 * 2^-7 of S, the sum of the magnitudes of the down product's terms; that sum's own fp32 rounding n 2^-24 S; the
route weights' 2e-5 S."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CASES = {
    "wide output, one token": dict(T=1, D=7168, F=256, E=4, K=2),
    "wide output, shared": dict(T=9, D=7168, F=512, E=4, K=2, Fs=2048),
    "wide output, 64 tokens": dict(T=64, D=7168, F=384, E=3, K=1),
    "wide experts, one token": dict(T=1, D=1024, F=14336, E=2, K=1),
    "wide experts, 17 tokens": dict(T=17, D=512, F=14336, E=2, K=2),
    "wide experts, bf16": dict(T=3, D=520, F=14344, E=2, K=1, fp8=False),
    "both wide, bf16": dict(T=2, D=7176, F=4104, E=2, K=2, fp8=False, Fs=14336),
    "both wide, clamped": dict(T=33, D=4096, F=14336, E=2, K=1, limit=1.0),
}


@pytest.mark.parametrize("name", CASES)
def test_against_the_formula(name):
    from mlops_b200 import layer, ops

    case = dict(dict(fp8=True, Fs=0, limit=None), **CASES[name])
    T, D, F, E, K, Fs, limit = (case[k] for k in ("T", "D", "F", "E", "K", "Fs", "limit"))
    g = torch.Generator(device=DEV).manual_seed(T + D)
    new = lambda *shape, std=1.0: torch.randn(*shape, generator=g, device=DEV).mul_(std).bfloat16()  # noqa: E731
    x, residual, router = new(T, D), new(T, D), new(E, D, std=2.0 / D ** 0.5)
    weights = [new(E, 2 * F, D, std=1.5 / D ** 0.5), new(E, D, F, std=1.5 / F ** 0.5)]
    shared = (new(2 * Fs, D, std=1.5 / D ** 0.5), new(D, Fs, std=1.5 / Fs ** 0.5)) if Fs else None
    values = weights
    if case["fp8"]:
        weights = [ops.quantize_blocks(w) for w in weights]
        values = [q.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2) for q, s in weights]
    call = lambda: layer.forward_decode(x, residual, router, *weights, top_k=K, routing_mode="softmax_then_topk",  # noqa: E731
                                        swiglu_limit=limit, shared=shared)
    output, share, ids = call()
    assert all(torch.equal(a, b) for a, b in zip(call(), (output, share, ids)))
    ops.check_status(DEV)

    logits = x.double() @ router.double().t()
    top = logits.sort(dim=-1, descending=True, stable=True)
    near = top.values[:, :K + 1]
    assert near.shape[1] == 1 or float((near[:, :-1] - near[:, 1:]).min()) > 1e-5, "choose another seed"
    expected_ids = top.indices[:, :K]
    expected_share = torch.softmax(logits, -1).gather(1, expected_ids)
    assert torch.equal(ids.long(), expected_ids) and float((share.double() / expected_share - 1).abs().max()) < 2e-5

    out, size = residual.double(), torch.zeros(T, D, dtype=torch.float64, device=DEV)
    terms = [(values[0][e], values[1][e], (expected_share * (expected_ids == e)).sum(1)) for e in range(E)]
    if shared is not None:
        terms.append((*shared, torch.ones(T, dtype=torch.float64, device=DEV)))
    for w13, w2, part in terms:
        gate, up = (x.double() @ w13.double().t()).chunk(2, -1)
        if limit is not None:
            gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        act = (gate * torch.sigmoid(gate) * up).bfloat16().double() * part[:, None]
        out += act @ w2.double().t()
        size += act.abs() @ w2.double().abs().t()
    tolerance = 2.0 ** -8 * out.abs() + (0.02 * 2.0 ** -7 + (K * F + Fs + 128) * 2.0 ** -24 + 4e-5) * size + 1e-30
    off = (output.double() - out).abs()
    assert bool((off <= tolerance).all()), float((off / tolerance).max())
