"""The layer for a few tokens (`layer.forward_decode`) against the same formula in 64 bits.

Tolerance of an output. Its own rounding to bf16: half a step, 2^-8 of the value. The activation's rounding to
bf16 is part of the formula, but the fp32 sums before it (relative error near sqrt(D) * 2^-24 * sum|x w| / |h|, 1e-5 at
the widest here, against a step of 2^-7) let under 1% of the activations round the other way; twice that, all with one
sign: 0.02 * 2^-7 of S, the sum of the magnitudes of the down product's terms. The fp32 sum of n terms: n * 2^-24 S."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _modules():
    from mlops_b200 import layer, ops

    return layer, ops


def _inputs(T, D, F, E, K, mode="softmax_then_topk", Fs=0, fp8=True, limit=None, seed=0, groups=1, kept=1, scaling=1.0,
            router_dtype=torch.float32, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    new = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16()  # noqa: E731
    s = dict(T=T, D=D, F=F, E=E, K=K, mode=mode, limit=limit, groups=groups, kept=kept, scaling=scaling,
             x=new(T, D), residual=new(T, D), bias=None, shared=None)
    s["router"] = (torch.randn(E, D, generator=g) * 2.0 / D ** 0.5).to(router_dtype)
    if skew:  # every token prefers the first experts
        s["x"][:, 0] = 1.0
        s["router"][:, 0] = -skew * torch.arange(E)
    if mode == "sigmoid_noaux_tc":
        s["bias"] = torch.randn(E, generator=g) * 0.1
    s["weights"], s["values"] = [], []
    for out, inner in ((2 * F, D), (D, F)):
        w = new(E, out, inner, std=1.5 / inner ** 0.5)
        if fp8:
            scale = (torch.rand(E, out // 128, inner // 128, generator=g) + 0.5) * 0.01 / inner ** 0.5
            wide = scale.repeat_interleave(128, 1).repeat_interleave(128, 2)
            q = (w.float() / wide).clamp(-448, 448).to(torch.float8_e4m3fn)
            s["weights"].append((q, scale))
            s["values"].append(q.double() * wide.double())
        else:
            s["weights"].append(w)
            s["values"].append(w.double())
    if Fs:
        s["shared"] = (new(2 * Fs, D, std=1.5 / D ** 0.5), new(D, Fs, std=1.5 / Fs ** 0.5))
    return s


def _call(s, **changes):
    layer, _ = _modules()
    dev = lambda t: t if t is None else tuple(u.to(DEV) for u in t) if isinstance(t, tuple) else t.to(DEV)  # noqa: E731
    kwargs = dict(top_k=s["K"], routing_mode=s["mode"], router_bias=dev(s["bias"]), n_group=s["groups"],
                  topk_group=s["kept"], routed_scaling=s["scaling"], swiglu_limit=s["limit"], shared=dev(s["shared"]))
    kwargs.update(changes)
    return layer.forward_decode(dev(s["x"]), dev(s["residual"]), dev(s["router"]), dev(s["weights"][0]),
                                dev(s["weights"][1]), **kwargs)


def _route(s):
    """64-bit weights and ids, and the smallest gap between keys that decide."""
    logits = s["x"].double() @ s["router"].bfloat16().double().t()
    keys = logits
    if s["mode"] == "sigmoid_noaux_tc":
        scores = torch.sigmoid(logits)
        keys = scores + s["bias"].double()
        grouped = keys.view(s["T"], s["groups"], -1)
        best = grouped.topk(min(2, grouped.shape[-1]), -1).values.sum(-1)
        kept = torch.zeros_like(best).scatter_(1, best.topk(s["kept"], -1).indices, 1.0)
        keys = torch.where(kept[..., None] > 0, grouped, -torch.inf).view_as(keys)
    top = keys.sort(dim=-1, descending=True, stable=True)
    ids = top.indices[:, :s["K"]]
    near = top.values[:, :s["K"] + 1]
    gap = float((near[:, :-1] - near[:, 1:]).min()) if near.shape[1] > 1 else 1.0
    if s["mode"] == "sigmoid_noaux_tc":
        picked = scores.gather(1, ids)
        return picked / picked.sum(-1, keepdim=True) * s["scaling"], ids, gap
    if s["mode"] == "softmax_then_topk":
        return torch.softmax(logits, -1).gather(1, ids), ids, gap
    return torch.softmax(logits.gather(1, ids), -1), ids, gap


def _swiglu(h, limit):
    gate, up = h.chunk(2, -1)
    if limit is not None:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return (gate * torch.sigmoid(gate) * up).bfloat16().double()


def _formula(s, weights, ids):
    """The output in 64 bits and S."""
    x, out = s["x"].double(), s["residual"].double()
    size = torch.zeros_like(out)
    terms = [(s["values"][0][e], s["values"][1][e], (ids == e).any(1).nonzero()[:, 0],
              (weights * (ids == e)).sum(1)) for e in ids.unique().tolist()]
    if s["shared"] is not None:
        terms.append((s["shared"][0].double(), s["shared"][1].double(), torch.arange(s["T"]), torch.ones(s["T"]).double()))
    for w13, w2, tokens, share in terms:
        act = _swiglu(x[tokens] @ w13.t(), s["limit"]) * share[tokens][:, None]
        out[tokens] += act @ w2.t()
        size[tokens] += act.abs() @ w2.abs().t()
    return out, size


def _check(s, results):
    output, weights, ids = (t.cpu() for t in results)
    expected_weights, expected_ids, gap = _route(s)
    assert gap > 1e-5, "choose another seed: the selection hangs on a rounding"
    assert torch.equal(ids.long(), expected_ids)
    # fp32 logits are off by about sqrt(D) 2^-24 of sum|x w|, a weight by as much relative
    assert float((weights.double() / expected_weights - 1).abs().max()) < 2e-5
    out, size = _formula(s, expected_weights, expected_ids)
    terms = s["K"] * s["F"] + (s["shared"][1].shape[1] if s["shared"] else 0) + 64
    tolerance = 2.0 ** -8 * out.abs() + (0.02 * 2.0 ** -7 + (terms + 64) * 2.0 ** -24 + 4e-5) * size + 1e-30
    off = (output.double() - out).abs()
    assert bool((off <= tolerance).all()), float((off / tolerance).max())


CASES = {
    "one token": dict(T=1, D=256, F=128, E=8, K=2),
    "one expert": dict(T=3, D=128, F=128, E=1, K=1),
    "every expert": dict(T=5, D=256, F=128, E=4, K=4),
    "fine": dict(T=1, D=2048, F=768, E=32, K=8, seed=1),
    "fine, seven": dict(T=7, D=2048, F=768, E=32, K=8),
    "wide": dict(T=2, D=1024, F=3584, E=4, K=2, mode="topk_then_softmax"),
    "nine tokens": dict(T=9, D=384, F=256, E=16, K=4),
    "33 tokens": dict(T=33, D=640, F=384, E=8, K=3),
    "64 tokens on few experts": dict(T=64, D=512, F=256, E=4, K=2),
    "64 tokens on one expert each": dict(T=64, D=256, F=256, E=3, K=1, skew=9.0),
    "grouped": dict(T=4, D=1792, F=512, E=32, K=4, mode="sigmoid_noaux_tc", groups=8, kept=4, scaling=2.5, Fs=512),
    "grouped, 40 tokens": dict(T=40, D=896, F=256, E=64, K=6, mode="sigmoid_noaux_tc", groups=4, kept=2, scaling=2.5, Fs=328, seed=2),
    "shared beside one token": dict(T=1, D=256, F=128, E=8, K=1, Fs=8),
    "bf16": dict(T=6, D=512, F=256, E=8, K=2, fp8=False),
    "bf16, ragged": dict(T=5, D=1000, F=712, E=12, K=3, fp8=False, mode="topk_then_softmax", limit=1.0),
    "bf16, smallest": dict(T=1, D=8, F=8, E=2, K=1, fp8=False),
    "bf16, odd tail": dict(T=17, D=72, F=200, E=5, K=5, fp8=False, Fs=24),
    "bf16 router": dict(T=3, D=384, F=128, E=20, K=3, router_dtype=torch.bfloat16),
    "clamped": dict(T=4, D=512, F=256, E=8, K=2, limit=0.5, Fs=128),
    "24 tokens an expert": dict(T=48, D=1024, F=640, E=8, K=4, Fs=200),
    "one expert, 64 tokens": dict(T=64, D=1280, F=896, E=1, K=1),
    "bf16, 48 tokens an expert": dict(T=64, D=520, F=328, E=4, K=3, fp8=False),
    "256 experts in 8 groups": dict(T=6, D=256, F=128, E=256, K=8, mode="sigmoid_noaux_tc", groups=8, kept=4, scaling=2.5),
    "1000 experts": dict(T=2, D=128, F=128, E=1000, K=32, seed=3),
}


@pytest.mark.parametrize("name", CASES)
def test_against_the_formula(name):
    s = _inputs(**CASES[name])
    results = _call(s)
    _check(s, results)
    again = _call(s)
    assert all(torch.equal(a, b) for a, b in zip(results, again))


@pytest.mark.parametrize("T", range(1, 65, 3))
def test_every_number_of_tokens(T):
    s = _inputs(T=T, D=256, F=128, E=6, K=2, fp8=T % 2 == 0, seed=T)
    _check(s, _call(s))


def test_extreme_weights_and_tokens_stay_their_own():
    """E4M3's smallest and largest values; a token of zeros; a NaN token and a NaN weight reach nobody else."""
    s = _inputs(T=6, D=256, F=128, E=8, K=2, seed=5)
    for q, _scale in s["weights"]:
        q.view(torch.uint8)[:, :4] = torch.tensor([0x01, 0x7e, 0xfe, 0x81], dtype=torch.uint8)[None, :, None]
    s["values"] = [q.double() * sc.repeat_interleave(128, 1).repeat_interleave(128, 2).double()
                   for q, sc in s["weights"]]
    s["x"][2] = 0
    s["router"] += 0
    clean = _call(s)
    expected_weights, ids, _ = _route(s)
    ids[2], expected_weights[2] = torch.tensor([0, 1]), torch.tensor([1 / 8, 1 / 8], dtype=torch.float64)  # ties: lowest index
    assert torch.equal(clean[2].cpu().long(), ids)
    out, size = _formula(s, expected_weights, ids)
    tolerance = 2.0 ** -8 * out.abs() + (0.02 * 2.0 ** -7 + 500 * 2.0 ** -24 + 4e-5) * size + 1e-30
    assert bool(((clean[0].cpu().double() - out).abs() <= tolerance).all())
    assert torch.equal(clean[0][2].cpu(), s["residual"][2])
    s["x"][4, 100] = float("nan")
    dirty = _call(s)
    rest = [0, 1, 2, 3, 5]
    assert bool(dirty[0][4].isnan().all()) and torch.equal(dirty[0][rest], clean[0][rest])
    s["x"][4, 100] = 0
    victim = int(clean[2][0, 0])
    s["weights"][1][0].view(torch.uint8)[victim, 7, 3] = 0x7f  # one output column of one expert
    dirty = _call(s)
    hit = (dirty[2] == victim).any(1)
    assert bool(dirty[0][hit, 7].isnan().all()) and not bool(dirty[0][~hit].isnan().any())
    dirty[0][:, 7], clean[0][:, 7] = 0, 0
    assert torch.equal(dirty[0][rest], clean[0][rest])


def test_no_tokens_shapes_and_a_stream_of_its_own():
    layer, ops = _modules()
    s = _inputs(T=4, D=256, F=128, E=8, K=2)
    empty = dict(s, x=s["x"][:0], residual=s["residual"][:0])
    out, weights, ids = _call(empty)
    assert out.shape == (0, 256) and weights.shape == (0, 2) and ids.shape == (0, 2)
    plain = _call(s)
    shaped = _call(dict(s, x=s["x"].view(2, 2, 256), residual=s["residual"].view(2, 2, 256)))
    assert shaped[0].shape == (2, 2, 256) and torch.equal(shaped[0].view(4, 256), plain[0])
    wide = torch.zeros(4, 512, dtype=torch.bfloat16)
    wide[:, ::2] = s["x"]
    assert torch.equal(_call(dict(s, x=wide[:, ::2]))[0], plain[0])  # any strides
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = _call(s)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(plain, side))
    ops.set_cta_limit(37)  # fewer SMs: other cuts, the same sums
    try:
        few = _call(s)
    finally:
        ops.set_cta_limit(0)
    _check(s, few)


def test_captured_calls_replay_together_with_eager_ones():
    layer, _ = _modules()
    s = _inputs(T=8, D=1024, F=512, E=16, K=4, seed=8)
    dev = [s["router"].to(DEV), tuple(t.to(DEV) for t in s["weights"][0]), tuple(t.to(DEV) for t in s["weights"][1])]
    kwargs = dict(top_k=4, routing_mode="softmax_then_topk")
    inputs = [[torch.zeros(8, 1024, dtype=torch.bfloat16, device=DEV) for _ in range(2)] for _ in range(2)]
    layer.forward_decode(*inputs[0], *dev, **kwargs)
    torch.cuda.synchronize()
    graphs, outputs = [], []
    for x, residual in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(layer.forward_decode(x, residual, *dev, **kwargs))
        graphs.append(graph)
    expected = []
    for i, (x, residual) in enumerate(inputs):
        fresh = _inputs(T=8, D=1024, F=512, E=16, K=4, seed=20 + i)
        x.copy_(fresh["x"])
        residual.copy_(fresh["residual"])
        expected.append(layer.forward_decode(x, residual, *dev, **kwargs))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = layer.forward_decode(*inputs[0], *dev, **kwargs)
    torch.cuda.synchronize()
    for got, want in zip([*outputs, eager], [*expected, expected[0]]):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_agrees_with_the_grouped_layer():
    """Same routing to the bit on well separated logits; on bf16 experts the grouped layer rounds h13, act, the
    expert rows and the output to bf16: four half steps on values of the size of S's square root of terms."""
    layer, _ = _modules()
    for fp8 in (False, True):
        s = _inputs(T=16, D=512, F=256, E=8, K=2, fp8=fp8, seed=3)
        dev = lambda t: tuple(u.to(DEV) for u in t) if isinstance(t, tuple) else t.to(DEV)  # noqa: E731
        full = layer.forward_routed(dev(s["x"]), dev(s["residual"]), dev(s["router"]), dev(s["weights"][0]),
                                    dev(s["weights"][1]), top_k=2, routing_mode="softmax_then_topk")
        few = _call(s)
        assert torch.equal(full[6], few[2])
        off = (full[0].float() - few[0].float()).norm() / few[0].float().norm()
        # E4M3 activations (two roundings of 2^-4 at most, 2.6% rms each) against bf16 ones (2^-8)
        assert float(off) < (0.06 if fp8 else 4 * 2.0 ** -8)
