"""The pre-activation kept in 8 bits (`swiglu_save8`, `restore8`, `dswiglu_saved8`) against its definition on the
CPU and the formulas in 64 bits, and the layer that runs on it.

Tolerances. Codes and their scales are defined to the bit. A bf16 result is off by half a step, 2^-8 of the
value, and by the fp32 arithmetic before it: about ten roundings and an exponential of two units in the last
place, under 32 * 2^-24 of the product's factors taken without cancellation. A sum of n fp32 terms in any order is
off by at most n * 2^-24 of the sum of magnitudes; each term carries the same arithmetic."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP, ULP = 2.0 ** -8, 2.0 ** -24


def _ops():
    from mlops_b200 import ops

    return ops


def _rows(rows, width, seed, std=1.5):
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(rows, 2 * width, generator=g) * std).bfloat16()
    return h, (torch.randn(rows, width, generator=g) * 0.5).bfloat16(), torch.rand(rows, generator=g), \
        torch.randperm(rows, generator=g).to(torch.int32)


def _blocks(width):
    """Column ranges of the blocks, gate's then up's."""
    return [(half + c, min(half + c + 128, half + width)) for half in (0, width) for c in range(0, width, 128)]


def _kept(h):
    """Codes, scales and values by the definition (fp32 quotients; the product exact, rounded once)."""
    width = h.shape[1] // 2
    codes, scales = torch.zeros(h.shape, dtype=torch.int8), torch.empty(h.shape[0], len(_blocks(width)))
    values = torch.empty(h.shape)
    for i, (low, high) in enumerate(_blocks(width)):
        part = h[:, low:high].float()
        a = part.abs().amax(1, keepdim=True).clamp_min(1e-30)
        codes[:, low:high] = torch.round(part.double() * (torch.full_like(a, 127.0) / a).double()).to(torch.int8)
        scales[:, i:i + 1] = a / 127.0
        values[:, low:high] = codes[:, low:high].float() * scales[:, i:i + 1]
    return codes, scales, values


def _formula(values, r, score, limit):
    """64-bit results and the magnitudes that bound the fp32 arithmetic's error."""
    width = r.shape[1]
    gate, up, r, score = values[:, :width].double(), values[:, width:].double(), r.double(), score.double()[:, None]
    keep_gate = keep_up = torch.ones_like(gate)
    if limit is not None:
        keep_gate, keep_up = (gate <= limit).double(), (up.abs() <= limit).double()
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    sig = torch.sigmoid(gate)
    silu, act = gate * sig, gate * sig * up
    grad = torch.cat([score * r * up * (sig + silu * (1 - sig)) * keep_gate, score * r * silu * keep_up], 1)
    size = torch.cat([(score * r * up).abs() * (sig + silu.abs()), (score * r * silu).abs()], 1)
    return dict(dscore=(r * act).sum(1), dscore_size=(r * act).abs().sum(1), grad=grad, grad_size=size,
                act=score * act)


def _near(actual, expected, tolerance):
    off = (actual.double().cpu() - expected).abs()
    assert bool((off <= tolerance).all()), float((off - tolerance).max())


SIZES = [(1, 8), (3, 16), (5, 128), (2, 136), (33, 712), (130, 384), (7, 2048), (4740, 256), (9, 14336)]


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("limit", [None, 2.0])
def test_forward_keeps_the_codes_and_changes_no_result(rows, width, limit):
    ops = _ops()
    h, *_ = _rows(rows, width, rows + width)
    h[0, : min(width, 128)] = 0  # a block of zeros
    h[-1, width:] *= 1e-33  # below the smallest scale
    codes, scales, values = _kept(h)
    dev = h.to(DEV)
    for quantized, rounded in ((True, False), (False, True), (True, True), (False, False)):
        q, s, act, (got, got_scales) = ops.swiglu_save8(dev, limit=limit, quantized=quantized, rounded=rounded)
        assert torch.equal(got.cpu(), codes) and torch.equal(got_scales.cpu(), scales)
        if not (quantized or rounded):
            assert q is None and s is None and act is None
            continue
        q0, s0, act0 = ops.swiglu_quantize(dev, limit=limit, quantized=quantized, rounded=rounded)
        if quantized:
            assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)
        if rounded:
            assert torch.equal(act, act0)
    restored = ops.restore8((got, got_scales))
    assert torch.equal(restored.cpu(), values.bfloat16())
    # within half a step of the codes, and half a step of bf16
    for low, high in _blocks(width):
        a = h[:, low:high].double().abs().amax(1, keepdim=True).clamp_min(1e-30)
        off = (restored.cpu()[:, low:high].double() - h[:, low:high].double()).abs()
        assert bool((off <= a / 254 * (1 + 2 ** -20) + STEP * a).all())


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("limit", [None, 2.0])
def test_backward_from_the_codes(rows, width, limit):
    ops = _ops()
    h, r, weights, order = _rows(rows, width, 7 * rows + width)
    codes, scales, values = _kept(h)
    expected = _formula(values, r, weights[order.long()], limit)
    slack = 32 * ULP * expected["grad_size"]
    saved = (codes.to(DEV), scales.to(DEV))
    quantized = width % 128 == 0
    dscore, gq, gs, grad, act = ops.dswiglu_saved8(saved, r.to(DEV), weights.to(DEV), order.to(DEV), limit=limit,
                                                   quantized=quantized, rounded=True, scaled_activation=True)
    ops.check_status(DEV)
    _near(dscore, expected["dscore"], (width + 64) * ULP * expected["dscore_size"] + 1e-30)
    _near(grad, expected["grad"], STEP * expected["grad"].abs() + slack + 1e-37)
    _near(act, expected["act"], (STEP + 32 * ULP) * expected["act"].abs() + 1e-37)
    if quantized:
        for i, (low, high) in enumerate(_blocks(width)):
            scale = gs[:, i:i + 1].double().cpu()
            part, room = expected["grad"][:, low:high], slack[:, low:high]
            _near(scale, (part.abs().amax(1, keepdim=True) / 448).clamp_min(1e-12),
                  4 * ULP * scale + room.amax(1, keepdim=True) / 448)
            # half a step of E4M3 (2^-4 of a normal value, 2^-10 below), of a quotient the scale may shift
            tolerance = torch.maximum(part.abs() * 2.0 ** -4, scale * 2.0 ** -10) + 2 * room + 2 ** -18 * part.abs()
            _near(gq[:, low:high].float().cpu().double() * scale, part, tolerance)
    again = ops.dswiglu_saved8(saved, r.to(DEV), weights.to(DEV), order.to(DEV), limit=limit, quantized=quantized,
                               rounded=True, scaled_activation=True)
    assert torch.equal(again[0], dscore) and torch.equal(again[3], grad) and torch.equal(again[4], act)
    only = ops.dswiglu_saved8(saved, r.to(DEV), weights.to(DEV), order.to(DEV), limit=limit, quantized=False)
    assert torch.equal(only[0], dscore) and all(t is None for t in only[1:])


def test_the_gradient_is_the_slope():
    """Central differences of sum(score * r * silu(g) * u) in 64 bits at the kept values."""
    ops = _ops()
    h, r, weights, order = _rows(4, 128, 3)
    codes, scales, values = _kept(h)
    score = weights[order.long()].double()[:, None]

    def total(v):
        return (score * r.double() * torch.nn.functional.silu(v[:, :128]) * v[:, 128:]).sum(1)

    _, _, _, grad, _ = ops.dswiglu_saved8((codes.to(DEV), scales.to(DEV)), r.to(DEV), weights.to(DEV), order.to(DEV),
                                          quantized=False, rounded=True)
    for column in (0, 5, 127, 128, 200, 255):
        nudge = torch.zeros(4, 256, dtype=torch.float64)
        nudge[:, column] = 1e-5
        slope = (total(values.double() + nudge) - total(values.double() - nudge)) / 2e-5
        # the differences' own error: third derivative * 1e-10 and 64-bit cancellation, far below 1e-7
        _near(grad[:, column], slope, STEP * slope.abs() + 1e-6)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_a_value_that_is_none_comes_back_as_nan_alone(bad):
    ops = _ops()
    h, r, weights, order = _rows(3, 264, 5)
    h[1, 130] = bad  # second of three gate blocks (the last has 8 columns)
    *_, act, saved = ops.swiglu_save8(h.to(DEV), quantized=False, rounded=True)
    restored = ops.restore8(saved).cpu()
    assert bool(restored[1, 128:256].isnan().all())
    _, _, values = _kept(torch.where(h.isfinite(), h, 0))
    fine = torch.ones(h.shape, dtype=torch.bool)
    fine[1, 128:256] = False
    assert torch.equal(restored[fine], values.bfloat16()[fine])
    dscore, _, _, grad, _ = ops.dswiglu_saved8(saved, r.to(DEV), weights.to(DEV), order.to(DEV), quantized=False,
                                               rounded=True)
    assert bool(dscore[1].isnan()) and not bool(dscore[[0, 2]].isnan().any())
    assert bool(grad[1, 128:256].isnan().all()) and not bool(grad[[0, 2]].isnan().any())


def test_no_rows_pitches_and_a_stream_of_its_own():
    ops = _ops()
    empty = ops.swiglu_save8(torch.empty(0, 256, dtype=torch.bfloat16, device=DEV))
    assert empty[3][0].shape == (0, 256) and empty[3][1].shape == (0, 2)
    assert ops.restore8(empty[3]).shape == (0, 256)
    none = torch.empty(0, device=DEV)
    results = ops.dswiglu_saved8(empty[3], torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), none,
                                 torch.empty(0, dtype=torch.int32, device=DEV), rounded=True)
    assert results[0].shape == (0,) and results[3].shape == (0, 256)

    h, r, weights, order = _rows(37, 200, 9)
    wide_h = torch.full((37, 416), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide_h[:, 8:408] = h.to(DEV)
    wide_r = torch.full((37, 216), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide_r[:, 8:208] = r.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        *_, (codes, scales) = ops.swiglu_save8(wide_h[:, 8:408], quantized=False)
        wide_codes = torch.full((37, 424), 99, dtype=torch.int8, device=DEV)
        wide_codes[:, 8:408] = codes
        wide_scales = scales.t().contiguous().t()  # column-major
        got = ops.dswiglu_saved8((wide_codes[:, 8:408], wide_scales), wide_r[:, 8:208], weights.to(DEV),
                                 order.to(DEV), quantized=False, rounded=True, scaled_activation=True)
    torch.cuda.current_stream().wait_stream(stream)
    kept = _kept(h)
    assert torch.equal(codes.cpu(), kept[0]) and torch.equal(scales.cpu(), kept[1])
    plain = ops.dswiglu_saved8((codes, scales), r.to(DEV), weights.to(DEV), order.to(DEV), quantized=False,
                               rounded=True, scaled_activation=True)
    for a, b in zip(got, plain):
        assert (a is None and b is None) or torch.equal(a, b)


def test_an_order_entry_out_of_range_is_reported():
    ops = _ops()
    h, r, weights, order = _rows(6, 128, 2)
    saved = ops.swiglu_save8(h.to(DEV))[3]
    order[4] = 6
    ops.dswiglu_saved8(saved, r.to(DEV), weights.to(DEV), order.to(DEV))
    with pytest.raises(ops.NativeError, match="malformed"):
        ops.check_status(DEV)


# --------------------------------------------------------------------------------- the layer
def _layer_inputs(tokens=96, width=256, experts=8, inner=128, fp8=True, seed=0):
    ops = _ops()
    g = torch.Generator().manual_seed(seed)
    new = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16().to(DEV)  # noqa: E731
    w13, w2 = new(experts, 2 * inner, width, std=0.05), new(experts, width, inner, std=0.05)
    x, residual, dy = new(tokens, width), new(tokens, width), new(tokens, width)
    router = torch.randn(experts, width, generator=g).mul(0.05).to(DEV)
    if fp8:
        w13, w2 = ops.quantize_blocks(w13), ops.quantize_blocks(w2)
    return x, residual, router, w13, w2, dy


@pytest.mark.parametrize("mode", ["softmax_then_topk", "sigmoid_noaux_tc"])
@pytest.mark.parametrize("fp8", [True, False])
def test_the_layer_differs_in_what_it_keeps_only(fp8, mode):
    """Forward results bit for bit; the gradients are those of the steps on the kept form, in the one-call
    form and in the step-by-step form."""
    from mlops_b200 import layer

    ops = _ops()
    x, residual, router, w13, w2, dy = _layer_inputs(fp8=fp8)
    kwargs = dict(top_k=2, routing_mode=mode)
    plain = layer.forward_routed(x, residual, router, w13, w2, **kwargs, swiglu_limit=3.0)
    kept = layer.forward_routed(x, residual, router, w13, w2, **kwargs, swiglu_limit=3.0, saved="int8")
    for a, b in zip(plain[:10], kept[:10]):
        assert torch.equal(a, b)
    codes, scales, values = _kept(plain[10].cpu())
    assert torch.equal(kept[10][0].cpu(), codes) and torch.equal(kept[10][1].cpu(), scales)
    aux = torch.tensor(0.5, device=DEV)

    def backward():
        return layer.backward_routed(dy, aux, None, x, router, w13, w2, *kept[4:], **kwargs, swiglu_limit=3.0,
                                     weight_grad_dtype=torch.float32)

    grads = backward()
    ops.GEMM_TIMINGS = []  # the step-by-step form
    try:
        steps = backward()
        again = layer.forward_routed(x, residual, router, w13, w2, **kwargs, swiglu_limit=3.0, saved="int8")
    finally:
        ops.GEMM_TIMINGS = None
    assert all(torch.equal(a, b) for a, b in zip(grads, steps))
    assert torch.equal(again[0], kept[0]) and all(torch.equal(a, b) for a, b in zip(again[10], kept[10]))
    ops.check_status(DEV)

    # dW2 = (score * act)^T-products of the kept values: against 64 bits on the values the codes stand for
    _, _, _, _, _, weights, ids, order, offsets, slots, _ = kept
    r_rows = dy.float().cpu()[(order.cpu().long() // 2)]
    score = weights.cpu().reshape(-1)[order.cpu().long()]
    gate, up = values[:, :128].double().clamp(max=3.0), values[:, 128:].double().clamp(-3.0, 3.0)
    act = score.double()[:, None] * torch.nn.functional.silu(gate) * up
    for e in range(8):
        low, high = int(offsets[e]), int(offsets[e + 1])
        expected = r_rows[low:high].double().t() @ act[low:high]
        size = r_rows[low:high].double().abs().t() @ act[low:high].abs()
        # act rounded to bf16 once, exact products, fp32 sums
        _near(grads[4][e], expected, (STEP + (high - low + 64) * ULP) * size + 1e-30)


@pytest.mark.parametrize("shared", [False, True])
def test_the_provider_keeps_half_the_bytes(shared):
    from mlops_b200 import provider
    from mlops_b200.weights import BlockFP8Weight

    ops = _ops()
    x, residual, router, w13, w2, dy = _layer_inputs(tokens=64)
    w13, w2 = BlockFP8Weight(*w13), BlockFP8Weight(*w2)
    extra = {}
    if shared:
        g = torch.Generator().manual_seed(4)
        extra = dict(shared_w13=(torch.randn(256, 256, generator=g) * 0.05).bfloat16().to(DEV),
                     shared_w2=(torch.randn(256, 128, generator=g) * 0.05).bfloat16().to(DEV))
    leaves = [x, residual, router, w13, w2, *extra.values()]
    for leaf in leaves:
        leaf.requires_grad_(True)

    def step(kind):
        held = {}

        def pack(t):
            if type(t) is not BlockFP8Weight:  # (kept either way, and without a storage of its own)
                held[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t

        previous = provider.set_saved_activations(kind)
        try:
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
                out = provider.apply(x, residual, router, w13, w2, top_k=2, routing_mode="softmax_then_topk", **extra)
        finally:
            assert provider.set_saved_activations(previous) == kind
        return out, torch.autograd.grad(out[0], leaves, dy), sum(held.values())

    out, grads, held = step("bf16")
    out8, grads8, held8 = step("int8")
    assert all(torch.equal(a, b) for a, b in zip(out, out8))
    rows = 128 + (64 if shared else 0)
    assert held - held8 == rows * (2 * 2 * 128) - rows * (2 * 128 + 4 * 2)
    # the gradients differ by what keeping eight bits costs: half a step is 1/254 of a block's largest value,
    # under 4 rms here, so under 1.6% of the rms of g and u; silu' and u enter each once
    for a, b in zip(grads8, grads):
        assert float((a.float() - b.float()).norm() / b.float().norm()) < 4 * 0.016
    assert torch.equal(grads8[1], grads[1])
    with torch.no_grad():  # nothing is kept where nothing is differentiated
        provider.set_saved_activations("int8")
        try:
            plain = provider.apply(x, residual, router, w13, w2, top_k=2, routing_mode="softmax_then_topk", **extra)
        finally:
            provider.set_saved_activations("bf16")
    assert torch.equal(plain[0], out[0])
    ops.check_status(DEV)


def test_operators_keep_the_contract():
    from mlops_b200 import provider

    x, residual, router, w13, w2, dy = _layer_inputs(tokens=16)
    args = (x, residual, router, w13[0], w2[0], torch.empty(0, device=DEV), 2, "softmax_then_topk", 1, 1, 1.0, [16],
            "float32", torch.float32, None, [w13[1], w2[1]])
    # (the schema check does arithmetic on every input, which E4M3 tensors have no kernels for)
    tests = ("test_faketensor",)
    torch.library.opcheck(provider.moe_save8_fwd, (x.requires_grad_(True), *args[1:]),
                          test_utils=("test_autograd_registration", "test_aot_dispatch_dynamic", *tests))
    x = x.detach()
    kept = provider.moe_save8_fwd(*args)
    none = torch.empty(0, device=DEV)
    torch.library.opcheck(provider.moe_saved8_bwd,
                          (dy, none, none, x, router, w13[0], w2[0], *kept[4:], 2, "softmax_then_topk", [16],
                           torch.float32, None, True, True, True, [w13[1], w2[1]]), test_utils=tests)
    h = torch.randn(3, 5, 80, device=DEV).bfloat16().requires_grad_(True)
    torch.library.opcheck(provider.swiglu_save8, (h, None))
    act, codes, scales = provider.swiglu_save8(h, 2.0)
    torch.library.opcheck(provider.swiglu_saved8_bwd, (codes, scales, torch.randn_like(act), 2.0), test_utils=tests)
    assert torch.equal(act, provider.swiglu(h, 2.0))


def test_a_captured_step_replays():
    ops = _ops()
    h, r, weights, order = (t.to(DEV) for t in _rows(300, 256, 21))

    def step():
        *_, saved = ops.swiglu_save8(h)
        return ops.dswiglu_saved8(saved, r, weights, order, rounded=True, scaled_activation=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    h.copy_(_rows(300, 256, 22)[0])
    graph.replay()
    eager = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                           b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
               for a, b in zip(results, eager))
