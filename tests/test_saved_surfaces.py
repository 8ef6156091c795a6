"""Which surfaces the setting of the kept form reaches: `provider.apply`, its shared expert included, and no other."""

import pytest
import torch

from mlops_b200 import composed, provider


@pytest.fixture
def calls(monkeypatch):
    """The operators behind `apply` replaced by recorders; the shared expert's library products run on the CPU."""
    seen = []

    def activation(h13, limit):
        gate, up = h13.chunk(2, -1)
        return torch.nn.functional.silu(gate) * up

    def forward(name, results):
        def call(h2, *_):
            seen.append(name)
            return tuple(h2 if i == 0 else None for i in range(results))
        return call

    monkeypatch.setattr(provider, "refusal", lambda *args, **kwargs: None)
    monkeypatch.setattr(provider, "swiglu", lambda h, limit: (seen.append("swiglu"), activation(h, limit))[1])
    monkeypatch.setattr(provider, "swiglu_save8", lambda h, limit: (seen.append("swiglu_save8"), (activation(h, limit),))[1])
    monkeypatch.setattr(provider, "moe_fwd", forward("moe_fwd", 11))
    monkeypatch.setattr(provider, "moe_save8_fwd", forward("moe_save8_fwd", 12))
    monkeypatch.setattr(composed, "prepare_fwd", forward("prepare", 10))
    monkeypatch.setattr(composed, "finish_fwd", forward("finish", 1))
    monkeypatch.setattr(composed.provider, "register_container", lambda cls: None)
    return seen


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_the_two_region_form_keeps_bf16_whatever_the_setting(calls, kind):
    new = lambda *shape: torch.randn(*shape).bfloat16()  # noqa: E731
    x, experts = new(4, 16), new(2, 16, 16)
    kwargs = dict(top_k=1, routing_mode="softmax_then_topk", shared_w13=new(16, 16).requires_grad_(True),
                  shared_w2=new(16, 8))
    previous = provider.set_saved_activations(kind)
    try:
        composed.apply(x, x, new(2, 16), experts, experts, **kwargs)
        assert calls == ["swiglu", "prepare", "finish"]
        calls.clear()
        provider.apply(x, x, new(2, 16), experts, experts, **kwargs)
        assert calls == (["swiglu", "moe_fwd"] if kind == "bf16" else ["swiglu_save8", "moe_save8_fwd"])
        calls.clear()
        with torch.no_grad():
            provider.apply(x, x, new(2, 16), experts, experts, **kwargs)
        assert calls == ["swiglu", "moe_fwd"]
    finally:
        provider.set_saved_activations(previous)
