"""Values that are none beside a clamp: what comes out of a NaN, or of a kept block that a NaN or an infinity made
unreadable, is a NaN, and never the clamp's border. Comparisons are exact: everything else keeps its bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ops():
    from mlops_b200 import ops

    return ops


def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _same(a, b):
    return torch.equal(_bits(a), _bits(b))


@pytest.mark.parametrize("limit", [2.0, 1e30])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("width,quantized", [(264, False), (384, True)])
def test_the_clamped_backward_of_an_unreadable_block_is_nan(width, quantized, bad, half, limit):
    """One value of the middle block of a half is none: its 128 columns are not known any more, nor which of them the
    clamp would have cut. Their activation, both halves' gradients and the row's dscore are NaN; where the other half's
    own value, which is known, is cut, its gradient is the 0 it always is."""
    ops = _ops()
    g = torch.Generator().manual_seed(width)
    h = (torch.randn(3, 2 * width, generator=g) * 1.5).bfloat16().to(DEV)
    r = (torch.randn(3, width, generator=g) * 0.5).bfloat16().to(DEV)
    weights, order = torch.rand(3, generator=g).to(DEV), torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)
    h[1, half * width + 130] = 0

    def backward():
        saved = ops.swiglu_save8(h, limit=limit, quantized=False)[3]
        results = ops.dswiglu_saved8(saved, r, weights, order, limit=limit, quantized=quantized, rounded=True,
                                     scaled_activation=True)
        return saved, results

    clean_saved, clean = backward()
    h[1, half * width + 130] = bad
    saved, (dscore, gq, gs, grad, act) = backward()
    ops.check_status(DEV)
    lost = torch.zeros(3, 2 * width, dtype=torch.bool, device=DEV)
    lost[1, half * width + 128:half * width + 256] = True
    assert torch.equal(ops.restore8(saved).isnan(), lost)
    columns = lost[:, :width] | lost[:, width:]
    codes, scales = clean_saved
    blocks = scales.shape[1] // 2
    wide = [scales[:, i * blocks:(i + 1) * blocks].repeat_interleave(128, 1)[:, :width] for i in (0, 1)]
    values = codes.float() * torch.cat(wide, 1)  # as they are kept, in fp32
    cut = torch.cat([values[:, :width] > limit, values[:, width:].abs() > limit], 1) & ~lost
    both = torch.cat([columns, columns], 1) & ~cut
    assert bool(dscore[1].isnan()) and torch.equal(dscore[[0, 2]], clean[0][[0, 2]])
    assert torch.equal(act.isnan(), columns) and _same(act[~columns], clean[4][~columns])
    assert torch.equal(grad.isnan(), both), (grad.isnan() != both).nonzero().tolist()
    assert _same(grad[~both], clean[3][~both])
    if quantized:
        assert torch.equal(gq.float().isnan(), both) and _same(gq[~both], clean[1][~both])
        kept = ~torch.cat([columns, columns], 1)[:, ::128]
        assert torch.equal(gs[kept], clean[2][kept])


@pytest.mark.parametrize("where", ["gate", "up", "shared gate", "shared up"])
@pytest.mark.parametrize("fp8", [True, False])
def test_a_nan_weight_of_the_up_product_reaches_its_tokens_through_the_clamp(fp8, where):
    """`layer.forward_decode` with a limit: one NaN in a gate or up row of an expert (of the shared expert) makes one
    activation NaN, and with it every output of the expert's tokens (of all); the others keep their bits."""
    from mlops_b200 import layer

    ops = _ops()
    g = torch.Generator().manual_seed(11)
    new = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).bfloat16().to(DEV)  # noqa: E731
    x, residual, router = new(11, 256), new(11, 256), new(8, 256, std=0.1)
    w13, w2, shared = new(8, 256, 256, std=0.1), new(8, 256, 128, std=0.1), (new(256, 256, std=0.1), new(256, 128, std=0.1))
    if fp8:
        w13, w2 = ops.quantize_blocks(w13), ops.quantize_blocks(w2)
    call = lambda: layer.forward_decode(x, residual, router, w13, w2, top_k=2, routing_mode="softmax_then_topk",  # noqa: E731
                                        swiglu_limit=0.5, shared=shared)
    clean, _, ids = call()
    assert not bool(clean.isnan().any())
    row = 77 + (128 if "up" in where else 0)
    if "shared" in where:
        shared[0][row, 3] = float("nan")
        hit = torch.ones(11, dtype=torch.bool, device=DEV)
    else:
        if fp8:
            w13[0].view(torch.uint8)[5, row, 3] = 0x7f
        else:
            w13[5, row, 3] = float("nan")
        hit = (ids == 5).any(1)
        assert 0 < int(hit.sum()) < 11
    output, _, again = call()
    assert torch.equal(again, ids) and bool(output[hit].isnan().all()) and torch.equal(output[~hit], clean[~hit])
    ops.check_status(DEV)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("save8", [False, True])
def test_the_clamped_activation_of_a_nan_is_nan(save8, half):
    """`swiglu_quantize` and `swiglu_save8` with a limit, to E4M3 and to bf16: the element alone, as without a limit."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    h = (torch.randn(5, 512, generator=g) * 1.5).bfloat16().to(DEV)
    call = lambda: (ops.swiglu_save8 if save8 else ops.swiglu_quantize)(h, limit=0.75, rounded=True)[:3]  # noqa: E731
    h[2, half * 256 + 140] = 0
    clean_q, clean_scales, clean = call()
    h[2, half * 256 + 140] = float("nan")
    q, scales, act = call()
    lost = torch.zeros(5, 256, dtype=torch.bool, device=DEV)
    lost[2, 140] = True
    # an activation of 0 (gate or up 0) is never its block's largest: the scales stay
    assert torch.equal(act.isnan(), lost) and torch.equal(act[~lost], clean[~lost])
    assert torch.equal(q.float().isnan(), lost) and _same(q[~lost], clean_q[~lost]) and torch.equal(scales, clean_scales)


@pytest.mark.parametrize("half", [0, 1])
def test_the_clamped_backward_of_a_nan_is_nan_but_for_what_is_cut(half):
    """`dswiglu_routed` with a limit: dscore and the activation are NaN, and so is the gradient of the half that holds a
    finite value; a NaN lies outside the clamp's range, so its own gradient is 0, as torch's clamp gives it."""
    ops = _ops()
    g = torch.Generator().manual_seed(4)
    h = torch.randn(4, 256, generator=g).clamp(-0.7, 0.7).bfloat16().to(DEV)  # nothing else is cut
    r, weights = torch.randn(4, 128, generator=g).bfloat16().to(DEV), torch.rand(4, generator=g).to(DEV)
    order = torch.arange(4, dtype=torch.int32, device=DEV)
    call = lambda: ops.dswiglu_routed(h, r, weights, order, limit=0.75, rounded=True, scaled_activation=True)  # noqa: E731
    clean = call()
    h[1, half * 128 + 9] = float("nan")
    dscore, _, _, grad, act = call()
    value = h.float().requires_grad_(True)
    gate, up = value[:, :128].clamp(max=0.75), value[:, 128:].clamp(-0.75, 0.75)
    expected = gate * torch.sigmoid(gate) * up
    slope, = torch.autograd.grad((weights[:, None] * r.float() * expected).sum(), value)
    other = torch.zeros(4, 256, dtype=torch.bool, device=DEV)
    other[1, (1 - half) * 128 + 9] = True
    assert torch.equal(slope.isnan(), other) and torch.equal(grad.isnan(), other) and float(grad[1, half * 128 + 9]) == 0.0
    changed = other | h.isnan()
    assert torch.equal(grad[~changed], clean[3][~changed])
    assert bool(dscore[1].isnan()) and torch.equal(dscore[[0, 2, 3]], clean[0][[0, 2, 3]])
    assert torch.equal(act.isnan(), h.isnan()[:, :128] | h.isnan()[:, 128:])


def test_the_fused_up_projection_clamps_a_nan_like_the_two_calls():
    ops = _ops()
    g = torch.Generator().manual_seed(6)
    x = torch.randn(40, 256, generator=g).bfloat16().to(DEV)
    w, ws = ops.quantize_blocks((torch.randn(2, 512, 256, generator=g) * 0.1).bfloat16().to(DEV))
    w.view(torch.uint8)[0, 30, 7] = 0x7f  # a gate row and an up row of the first group
    w.view(torch.uint8)[0, 256 + 99, 8] = 0x7f
    xq, xs = ops.quantize_rows(x)
    offsets = torch.tensor([0, 23, 40], dtype=torch.int32, device=DEV)
    h13 = ops.grouped_gemm_fp8(xq, xs, w, ws, offsets)
    q, scales, act = ops.swiglu_quantize(h13, limit=0.5, rounded=True)
    fused_h13, fused_q, fused_scales = ops.grouped_gemm_fp8_swiglu(xq, xs, w, ws, offsets, limit=0.5)
    ops.check_status(DEV)
    lost = torch.zeros(40, 256, dtype=torch.bool, device=DEV)
    lost[:23, 30] = lost[:23, 99] = True
    assert torch.equal(act.isnan(), lost) and torch.equal(q.float().isnan(), lost)
    assert _same(fused_q, q) and torch.equal(fused_scales, scales)
    assert torch.equal(fused_h13.view(torch.int16)[~h13.isnan()], h13.view(torch.int16)[~h13.isnan()])
