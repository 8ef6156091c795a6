"""Two operators around the expert products, as timed cases.

`case["path"]`:
  decode    the whole routed layer for a few tokens, one step of a serving loop: router, expert selection, up
            product, SwiGLU, down product and the weighted sum, with the shared expert where the layer has one
            (`layer.forward_decode`)
  save      SwiGLU of a training step's forward pass that keeps the pre-activation in 8 bits, and what the
            kept form stands for (`ops.swiglu_save8`, `ops.restore8`)
  saved     the routed SwiGLU backward from the kept 8 bits (`ops.dswiglu_saved8`)

`own` selects the library's calls; without it the same results come from elementary torch operations in 32 bits
(64 where a selection or a rounding sits next to a border), rounded once at the end.
"""

import math

import torch

own = False

# D hidden width, F expert width, E experts, K experts per token: the layers the benchmark runs
SHAPES = {
    # the small layer of the CPU-runnable configuration
    "small": dict(D=256, F=512, E=8, K=2, mode="softmax_then_topk"),
    # few wide experts
    "wide": dict(D=4096, F=14336, E=8, K=2, mode="softmax_then_topk"),
    # many narrow experts
    "fine": dict(D=2048, F=768, E=128, K=8, mode="softmax_then_topk"),
    # group-limited sigmoid routing beside a shared expert
    "grouped": dict(D=7168, F=2048, E=256, K=8, mode="sigmoid_noaux_tc", n_group=8, topk_group=4, scaling=2.5,
                    shared=2048),
}
LAYER = dict(n_group=1, topk_group=1, scaling=1.0, shared=0, experts="fp8", limit=0.0)
WEIGHT_STD = 0.02
BIAS_STD = 0.1  # a trained selection bias


def _decode(shape, T, **changes):
    return dict(LAYER, path="decode", T=T, **{**SHAPES[shape], **changes})


def _save(rows, F, form, limit=0.0):
    return dict(path="save", rows=rows, F=F, form=form, limit=limit)


def _saved(rows, F, form, limit=0.0):
    return dict(path="saved", rows=rows, F=F, form=form, limit=limit)


def listed():
    return [
        # the next token of one sequence: the smallest call, latency and launches
        dict(_decode("fine", 1), name="decode_fine_1"),
        # the small layer, two sequences
        dict(_decode("small", 2), name="decode_small_2"),
        # one sequence on the 256-expert layer with its shared expert
        dict(_decode("grouped", 1), name="decode_grouped_1"),
        # a serving batch on it: nearly every expert's weights are read, for two tokens each
        dict(_decode("grouped", 64), name="decode_grouped_64"),
        # a full batch on many narrow experts
        dict(_decode("fine", 48), name="decode_fine_48"),
        # few wide experts, an odd batch of which every expert gets several tokens
        dict(_decode("wide", 17), name="decode_wide_17"),
        # experts kept in bf16, ragged widths (multiples of 8 only), clamped activations
        dict(_decode("fine", 5, experts="bf16", D=1000, F=712, E=24, K=3, mode="topk_then_softmax", limit=7.0),
             name="decode_bf16_ragged_5"),
        # a small micro-batch of the small layer: launch-bound
        dict(_save(1024, 512, "bf16"), name="save_small_1024"),
        # a training micro-batch on 256 experts (8192 tokens, 8 experts each): E4M3 operands for the down product
        dict(_save(65536, 2048, "fp8"), name="save_grouped_65536"),
        # bf16 experts of the wide layer, an odd number of rows
        dict(_saved(8198, 14336, "bf16"), name="saved_wide_8198"),
        # the 256-expert micro-batch's backward pass with every result
        dict(_saved(65536, 2048, "fp8"), name="saved_grouped_65536"),
        # a small odd one with clamped activations
        dict(_saved(1031, 712, "bf16", 7.0), name="saved_ragged_1031"),
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    path = rng.choices(["decode", "save", "saved"], weights=[5, 2, 3])[0]
    limit = rng.choice([0.0, 0.0, 0.0, 7.0])
    if path != "decode":
        form = rng.choice(["fp8", "bf16"])
        F = 128 * _spread(rng, 1, 112) if form == "fp8" else 8 * _spread(rng, 2, 1792)
        rows = _spread(rng, 1, max(2, (65536 * 2048) // max(F, 2048)))
        return _save(rows, F, form, limit) if path == "save" else _saved(rows, F, form, limit)
    shape = rng.choice(["small", "wide", "fine", "grouped", "other", "other"])
    T = _spread(rng, 1, 64)
    if shape != "other":
        changes = dict(E=rng.choice([64, 128])) if shape == "grouped" else {}
        return _decode(shape, T, limit=limit, **changes)
    experts = rng.choice(["fp8", "bf16"])
    step = 128 if experts == "fp8" else 8
    groups = rng.choice([1, 1, 2, 4])
    return _decode("fine", T, limit=limit, experts=experts, D=step * _spread(rng, 256 // step, 5120 // step),
                   F=step * _spread(rng, 128 // step, 2560 // step), E=rng.choice([8, 16, 32, 60]),
                   K=rng.choice([1, 2, 4, 6, 8]), n_group=groups, topk_group=rng.randint(1, groups),
                   shared=rng.choice([0, 0, 8 * _spread(rng, 16, 256)]),
                   mode=rng.choice(["softmax_then_topk", "topk_then_softmax"]) if groups == 1 else "sigmoid_noaux_tc")


# ------------------------------------------------------------------------------ inputs
def _randn(generator, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=generator, device="cuda", dtype=dtype).mul_(std)


def _weight(generator, kind, experts, out, inner):
    """`[E, out, in]` expert weights: bf16, or E4M3 data with one fp32 scale per 128 x 128 block."""
    if kind == "bf16":
        return _randn(generator, experts, out, inner, std=WEIGHT_STD)
    data = torch.empty((experts, out, inner), dtype=torch.float8_e4m3fn, device="cuda")
    step = max(1, (1 << 29) // (out * inner))
    for low in range(0, experts, step):
        part = _randn(generator, min(step, experts - low), out, inner, std=100.0)
        data[low:low + step] = part.clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    scale = torch.rand((experts, out // 128, inner // 128), generator=generator, device="cuda")
    return data, (scale + 0.5) * (WEIGHT_STD / 100.0)


def _pad_blocks(v):
    """`[rows, F]` as `[rows, ceil(F / 128), 128]`, zeros behind the last column."""
    rows, width = v.shape
    blocks = -(-width // 128)
    return torch.nn.functional.pad(v, (0, 128 * blocks - width)).view(rows, blocks, 128)


def _codes(h13):
    """The 8-bit form of `[gate | up]` rows: int8 codes and one fp32 scale per row, half and 128 columns."""
    rows, width = h13.shape[0], h13.shape[1] // 2
    halves = h13.reshape(2 * rows, width)
    blocks = _pad_blocks(halves).float()
    largest = blocks.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    factor = torch.full_like(largest, 127.0).div_(largest)  # (a number over a tensor is a reciprocal and a product)
    codes = torch.round(blocks.double() * factor.double()).to(torch.int8)
    codes = codes.view(2 * rows, -1)[:, :width].reshape(rows, 2 * width)
    return codes, (largest / 127.0).view(rows, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["path"] != "decode":
        rows, F = case["rows"], case["F"]
        h13 = _randn(g, rows, 2 * F, std=1.5)
        if case["path"] == "save":
            return dict(case=case, h13=h13)
        codes, scales = _codes(h13)
        return dict(case=case, codes=codes, scales=scales, r=_randn(g, rows, F, std=0.5),
                    weights=torch.rand(rows, generator=g, device="cuda"),
                    order=torch.randperm(rows, generator=g, device="cuda").to(torch.int32))
    D, F, E, T = case["D"], case["F"], case["E"], case["T"]
    state = dict(case=case, x=_randn(g, T, D), residual=_randn(g, T, D),
                 router=_randn(g, E, D, std=WEIGHT_STD, dtype=torch.float32), bias=None, shared=None,
                 w13=_weight(g, case["experts"], E, 2 * F, D), w2=_weight(g, case["experts"], E, D, F))
    if case["mode"] == "sigmoid_noaux_tc":
        state["bias"] = _randn(g, E, std=BIAS_STD, dtype=torch.float32)
    if case["shared"]:
        state["shared"] = (_randn(g, 2 * case["shared"], D, std=WEIGHT_STD), _randn(g, D, case["shared"], std=WEIGHT_STD))
    return state


# ------------------------------------------------------------------------- the plain form
def _silu(gate):
    return gate / (1.0 + torch.exp(-gate))


def _route(logits, case, bias):
    """`(weights, ids)` of 64-bit logits; ties go to the lowest index."""
    K, experts = case["K"], case["E"]
    if case["mode"] == "sigmoid_noaux_tc":
        scores = 1.0 / (1.0 + torch.exp(-logits))
        keys = scores + bias.double()
        groups = keys.view(-1, case["n_group"], experts // case["n_group"])
        best = groups.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices[:, :case["topk_group"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        keys = torch.where(kept[..., None], groups, -math.inf).view_as(keys)
        ids = keys.sort(dim=-1, descending=True, stable=True).indices[:, :K]
        picked = scores.gather(1, ids)
        return (picked / picked.sum(-1, keepdim=True) * case["scaling"]).float(), ids
    ids = logits.sort(dim=-1, descending=True, stable=True).indices[:, :K]
    over = logits.gather(1, ids) if case["mode"] == "topk_then_softmax" else logits
    largest = over.amax(-1, keepdim=True)
    total = torch.exp(over - largest).sum(-1, keepdim=True)
    return (torch.exp(logits.gather(1, ids) - largest) / total).float(), ids


def _values(weight, which):
    """fp32 values of the experts `which`."""
    if isinstance(weight, torch.Tensor):
        return weight[which].float()
    data, scale = weight
    values = data.view(torch.uint8)[which].view(torch.float8_e4m3fn).float()
    experts, out, inner = values.shape
    values.view(experts, out // 128, 128, inner // 128, 128).mul_(scale[which][:, :, None, :, None])
    return values


def _activation(h13, limit):
    gate, up = h13.chunk(2, -1)
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return _silu(gate) * up


def _plain_decode(s):
    case, x = s["case"], s["x"].float()
    logits = s["x"].double() @ s["router"].to(torch.bfloat16).double().t()
    weights, ids = _route(logits, case, s["bias"])
    share = torch.zeros(logits.shape, device=x.device).scatter_(1, ids, weights)  # [T, E]
    # the experts that can have a token: all of them, or as many as there are assignments
    which = (share != 0).sum(0).topk(min(case["E"], ids.numel())).indices
    act = _activation(torch.matmul(x, _values(s["w13"], which).transpose(1, 2)), case["limit"])
    act *= share.t()[which][:, :, None]
    output = s["residual"].float() + torch.matmul(act, _values(s["w2"], which).transpose(1, 2)).sum(0)
    if s["shared"] is not None:
        output += _activation(x @ s["shared"][0].float().t(), case["limit"]) @ s["shared"][1].float().t()
    return dict(output=output.to(torch.bfloat16), weights=weights, ids=ids.to(torch.int32))


def _e4m3(values):
    """E4M3 values with one fp32 scale per row and 128 columns."""
    blocks = values.view(values.shape[0], -1, 128)
    scale = (blocks.abs().amax(-1, keepdim=True) * (1.0 / 448.0)).clamp_min(1e-12)
    q = (blocks / scale).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(values.shape), scale[..., 0]


def _plain_save(s):
    case, h13 = s["case"], s["h13"]
    rows, width = h13.shape[0], case["F"]
    codes, scales = _codes(h13)
    restored = _pad_blocks(codes.view(2 * rows, width)).float() * scales.view(2 * rows, -1, 1)
    restored = restored.view(2 * rows, -1)[:, :width].reshape(rows, 2 * width)
    act = _activation(h13.float(), case["limit"])
    found = dict(restored=restored.to(torch.bfloat16))
    if case["form"] == "fp8":
        found["act"], found["act_scales"] = _e4m3(act)
    else:
        found["act"] = act.to(torch.bfloat16)
    return found


def _slopes(gate, up, limit):
    """silu(gate), its slope, up, and where a gradient goes through (none through a clamped value)."""
    through_gate = through_up = 1.0
    if limit:
        through_gate, through_up = gate <= limit, up.abs() <= limit
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    sigmoid = 1.0 / (1.0 + torch.exp(-gate))
    silu = gate * sigmoid
    return silu, (sigmoid + silu * (1.0 - sigmoid)) * through_gate, up, through_up


def _plain_saved(s):
    case = s["case"]
    rows, width = s["r"].shape
    h13 = _pad_blocks(s["codes"].view(2 * rows, width)).float() * s["scales"].view(2 * rows, -1, 1)
    h13 = h13.view(2 * rows, -1)[:, :width].reshape(rows, 2 * width)
    silu, slope, up, through = _slopes(h13[:, :width], h13[:, width:], case["limit"])
    r, score = s["r"].float(), s["weights"][s["order"].long()][:, None]
    act = silu * up
    grad = torch.cat([score * r * up * slope, score * r * silu * through], 1)
    found = dict(dscore=(r * act).sum(-1, dtype=torch.float64).float(), grad=grad.to(torch.bfloat16),
                 act=(score * act).to(torch.bfloat16))
    if case["form"] == "fp8":
        found["grad_q"], found["grad_scales"] = _e4m3(grad)
    return found


# ------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return {"decode": _plain_decode, "save": _plain_save, "saved": _plain_saved}[case["path"]](state)
    from mlops_b200 import layer, ops

    limit = case["limit"] or None
    quantized = case.get("form") == "fp8"
    if case["path"] == "decode":
        output, weights, ids = layer.forward_decode(
            state["x"], state["residual"], state["router"], state["w13"], state["w2"], top_k=case["K"],
            routing_mode=case["mode"], router_bias=state["bias"], n_group=case["n_group"],
            topk_group=case["topk_group"], routed_scaling=case["scaling"], swiglu_limit=limit, shared=state["shared"])
        return dict(output=output, weights=weights, ids=ids)
    if case["path"] == "save":
        act_q, act_scales, act, saved = ops.swiglu_save8(state["h13"], limit=limit, quantized=quantized,
                                                         rounded=not quantized)
        found = dict(restored=ops.restore8(saved))
        return dict(found, act=act_q, act_scales=act_scales) if quantized else dict(found, act=act)
    dscore, grad_q, grad_scales, grad, act = ops.dswiglu_saved8(
        (state["codes"], state["scales"]), state["r"], state["weights"], state["order"], limit=limit,
        quantized=quantized, rounded=True, scaled_activation=True)
    found = dict(dscore=dscore, grad=grad, act=act)
    return dict(found, grad_q=grad_q, grad_scales=grad_scales) if quantized else found


# --------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Bytes: each input read once (of the experts, those that get a token), each output and the kept
    form written once. FLOPs: the products."""
    if case["path"] != "decode":
        rows, F, fp8 = case["rows"], case["F"], case["form"] == "fp8"
        kept = rows * (2 * F + 8 * -(-F // 128))
        if case["path"] == "save":
            return dict(bytes=4 * rows * F + kept + 4 * rows * F + rows * F * (1.03125 if fp8 else 2), flops=0)
        return dict(bytes=kept + 2 * rows * F + 12 * rows + 6 * rows * F + (rows * F * 2.0625 if fp8 else 0), flops=0)
    D, F, E, T, K = case["D"], case["F"], case["E"], case["T"], case["K"]
    active = E * (1 - (1 - K / E) ** T)  # expected number of experts that get a token
    nbytes = active * 3 * D * F * (2 if case["experts"] == "bf16" else 1) + 4 * E * D + 6 * T * D + 8 * T * K
    return dict(bytes=nbytes + 6 * D * case["shared"],
                flops=6 * T * K * D * F + 2 * T * E * D + 6 * T * D * case["shared"])


# --------------------------------------------------------------------- in 64 bits, written apart
def _exact_swiglu(gate, up, limit):
    if limit:
        gate = torch.minimum(gate, torch.full_like(gate, limit))
        up = torch.maximum(torch.minimum(up, torch.full_like(up, limit)), torch.full_like(up, -limit))
    return gate * up * torch.special.expit(gate)


def _exact_choice(logits, case, bias):
    """Route weights and ids, token by token on the host."""
    weights, ids = [], []
    for t, row in enumerate(logits.cpu().tolist()):
        if case["mode"] == "sigmoid_noaux_tc":
            score = [1.0 / (1.0 + math.exp(-v)) for v in row]
            key = [a + b for a, b in zip(score, bias)]
            size = len(row) // case["n_group"]
            rank = sorted(range(case["n_group"]),
                          key=lambda j: (-sum(sorted(key[j * size:(j + 1) * size])[-2:]), j))[:case["topk_group"]]
            allowed = [e for e in range(len(row)) if e // size in rank]
        else:
            score, key, allowed = None, row, range(len(row))
        mine = sorted(allowed, key=lambda e: (-key[e], e))[:case["K"]]
        if score is not None:
            total = math.fsum(score[e] for e in mine)
            weights.append([score[e] / total * case["scaling"] for e in mine])
        else:
            top = max(row)
            total = math.fsum(math.exp(v - top) for v in (row if case["mode"] == "softmax_then_topk"
                                                          else [row[e] for e in mine]))
            weights.append([math.exp(row[e] - top) / total for e in mine])
        ids.append(mine)
    return weights, ids


def _exact_matrix(weight, e):
    if isinstance(weight, torch.Tensor):
        return weight[e].double()
    wide = weight[1][e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    return weight[0][e].to(torch.float32).double() * wide


def exact(case, seed):
    s = prepare(case, seed)
    limit = case["limit"]
    if case["path"] == "decode":
        x, F = s["x"].double(), case["F"]
        logits = x @ s["router"].to(torch.bfloat16).double().t()
        weights, ids = _exact_choice(logits, case, None if s["bias"] is None else s["bias"].tolist())
        output = s["residual"].double()
        for e in sorted({e for row in ids for e in row}):
            tokens = [t for t, row in enumerate(ids) if e in row]
            share = torch.tensor([weights[t][ids[t].index(e)] for t in tokens], dtype=torch.float64, device=x.device)
            h = x[tokens] @ _exact_matrix(s["w13"], e).t()
            output[tokens] += share[:, None] * (_exact_swiglu(h[:, :F], h[:, F:], limit) @ _exact_matrix(s["w2"], e).t())
        if s["shared"] is not None:
            h = x @ s["shared"][0].double().t()
            half = case["shared"]
            output += _exact_swiglu(h[:, :half], h[:, half:], limit) @ s["shared"][1].double().t()
        return dict(output=output, weights=torch.tensor(weights, dtype=torch.float64), ids=None)
    rows, F = case["rows"], case["F"]
    pieces = []
    for low in range(0, rows, 4096):  # a slice of rows at a time: 64 bits of everything is large
        part = slice(low, min(rows, low + 4096))
        if case["path"] == "save":
            h = s["h13"][part].double()
            found = dict(act=_exact_swiglu(h[:, :F], h[:, F:], limit), restored=torch.empty_like(h))
            for c in [half + c for half in (0, F) for c in range(0, F, 128)]:
                stop = min(c + 128, F if c < F else 2 * F)
                block = s["h13"][part, c:stop]
                top = block.abs().amax(1, keepdim=True).float().clamp_min(1e-30)
                # the kept form is defined by its two fp32 factors; the codes are whole numbers
                codes = torch.round(block.double() * (torch.full_like(top, 127.0) / top).double())
                found["restored"][:, c:stop] = codes * torch.div(top, 127.0).double()
            names = ["act"] if case["form"] == "fp8" else []
        else:
            scales, codes = s["scales"][part].double(), s["codes"][part].double()
            blocks = scales.shape[1] // 2
            gate = codes[:, :F] * scales[:, :blocks].repeat_interleave(128, 1)[:, :F]
            up = codes[:, F:] * scales[:, blocks:].repeat_interleave(128, 1)[:, :F]
            r = s["r"][part].double()
            score = s["weights"][s["order"][part].long()].double()[:, None]
            act = _exact_swiglu(gate, up, limit)
            cut_gate, cut_up = (gate > limit, up.abs() > limit) if limit else (None, None)
            if limit:
                gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
            sig = torch.special.expit(gate)
            dgate = score * r * up * sig * (1.0 + gate * (1.0 - sig))
            dup = score * r * gate * sig
            if limit:
                dgate[cut_gate], dup[cut_up] = 0.0, 0.0
            found = dict(dscore=(r * act).sum(1), grad=torch.cat([dgate, dup], 1), act=score * act)
            names = ["grad"] if case["form"] == "fp8" else []
        for name in names:  # E4M3 values and their scales
            v = found[name]
            scale = (v.abs().view(v.shape[0], -1, 128).amax(2) / 448.0).clamp_min(1e-12)
            q = (v / scale.repeat_interleave(128, 1)).to(torch.float8_e4m3fn).float().double()
            found.update({"act": q, "act_scales": scale} if name == "act" else {"grad_q": q, "grad_scales": scale})
        pieces.append(found)
    return {name: torch.cat([p[name] for p in pieces]) for name in pieces[0]}
