"""Group-limited routing whose kept groups hold fewer than K experts: the places left go to the excluded experts, lowest id
first, each with its own score, as a stable sort of selection values gives them whose excluded entries are -infinity."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _expected(logits, bias, K, groups, kept, scaling):
    """In 64 bits, token by token: the kept groups' experts by selection value, then the others by id."""
    scores = torch.sigmoid(logits.double())
    keys = scores + bias.double()
    size = logits.shape[1] // groups
    ids = []
    for row in keys.tolist():
        best = [sum(sorted(row[g * size:(g + 1) * size])[-2:]) for g in range(groups)]
        chosen = sorted(range(groups), key=lambda g: (-best[g], g))[:kept]
        inside = sorted((e for e in range(len(row)) if e // size in chosen), key=lambda e: (-row[e], e))
        outside = [e for e in range(len(row)) if e // size not in chosen]
        ids.append((inside + outside)[:K])
    ids = torch.tensor(ids)
    picked = scores.gather(1, ids)
    return picked / picked.sum(1, keepdim=True) * scaling, ids


CASES = [(8, 4, 4, 1), (8, 8, 4, 1), (16, 6, 8, 2), (12, 5, 12, 3), (40, 32, 8, 2), (60, 20, 4, 1), (1024, 32, 32, 1)]


@pytest.mark.parametrize("experts,top_k,groups,kept", CASES)
def test_route_topk_fills_up(experts, top_k, groups, kept):
    from mlops_b200 import ops

    g = torch.Generator().manual_seed(experts + top_k)
    logits, bias = torch.randn(9, experts, generator=g), torch.randn(experts, generator=g) * 0.1
    weights, ids = ops.route_topk(logits.to(DEV), top_k, "sigmoid_noaux_tc", bias=bias.to(DEV), n_group=groups,
                                  topk_group=kept, routed_scaling=2.5)
    expected, expected_ids = _expected(logits, bias, top_k, groups, kept, 2.5)
    assert torch.equal(ids.cpu().long(), expected_ids)
    # a score: exponential of two units in the last place, a sum and a reciprocal; K summands; a quotient, a product
    assert float((weights.cpu().double() / expected - 1).abs().max()) < (top_k + 12) * 2.0 ** -23


def test_the_layer_for_a_few_tokens_fills_up():
    """Output: its own rounding 2^-8; act's, 2^-8 of each term, at most 2^-8 of S, the sum of the terms' magnitudes."""
    from mlops_b200 import layer

    g = torch.Generator().manual_seed(2)
    new = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16()  # noqa: E731
    T, D, F, E, K = 5, 256, 128, 8, 4
    x, residual, router, bias = new(T, D), new(T, D), new(E, D, std=0.1), torch.randn(E, generator=g) * 0.1
    w13, w2 = new(E, 2 * F, D, std=0.1), new(E, D, F, std=0.1)
    output, weights, ids = layer.forward_decode(
        *(t.to(DEV) for t in (x, residual, router, w13, w2)), top_k=K, routing_mode="sigmoid_noaux_tc",
        router_bias=bias.to(DEV), n_group=4, topk_group=1, routed_scaling=2.5)
    expected, expected_ids = _expected(x.double() @ router.double().t(), bias, K, 4, 1, 2.5)
    assert torch.equal(ids.cpu().long(), expected_ids)
    assert float((weights.cpu().double() / expected - 1).abs().max()) < 2e-5  # fp32 logits of 256 terms
    out, size = residual.double(), torch.zeros(T, D, dtype=torch.float64)
    for t in range(T):
        for k in range(K):
            e = int(expected_ids[t, k])
            gate, up = (w13[e].double() @ x[t].double()).chunk(2)
            act = float(expected[t, k]) * torch.nn.functional.silu(gate) * up
            out[t] += w2[e].double() @ act
            size[t] += w2[e].double().abs() @ act.abs()
    off = (output.cpu().double() - out).abs()
    assert bool((off <= 2.0 ** -8 * out.abs() + (2.0 ** -8 + 1e-4) * size).all())
