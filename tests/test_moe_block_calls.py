"""Calls of the MoE block on the CPU: the routed experts and the router are stand-ins, what is looked at is what the block asks of its
shared expert."""
import types

import pytest
import torch
from torch import nn


class _Routed(nn.Module):
    intermediate_size_per_partition = 16

    def forward(self, hidden_states, **kw):
        return torch.zeros_like(hidden_states)


class _Shared(nn.Module):
    """A shared expert of a user's own: rows in, rows out, no notion of adapters."""

    def __init__(self):
        super().__init__()
        self.down_proj = types.SimpleNamespace(input_size=16)

    def forward(self, x):
        return x + 1


def _block(shared, monkeypatch):
    from omni_infer_amd import config
    from omni_infer_amd.layers.deepseek_moe import DeepseekMoE
    monkeypatch.setattr(config.model_extra_config.operator_opt_config, "enable_moe_expert_parallel", False)
    b = DeepseekMoE.__new__(DeepseekMoE)
    nn.Module.__init__(b)
    b.experts, b.shared_experts, b.ep_size, b.fused, b.quant_symbol = _Routed(), shared, 1, False, False
    monkeypatch.setattr(DeepseekMoE, "_route", lambda self, h, m=None: (None, None))
    return b


@pytest.mark.parametrize("adapters", [None, object()])
def test_a_shared_expert_of_another_class(adapters, monkeypatch):
    b = _block(_Shared(), monkeypatch)
    x, res = torch.randn(3, 8), torch.randn(3, 8)
    kw = {} if adapters is None else {"adapters": adapters}   # a batch of adapters that the block has no room for
    y, r = b(x, res, None, 3, **kw)
    assert torch.equal(y, x + 1) and r is res


def test_no_shared_expert(monkeypatch):
    b = _block(None, monkeypatch)
    x = torch.randn(3, 8)
    assert torch.equal(b(x, None, None, 3, adapters=object())[0], torch.zeros(3, 8))


def test_bodies_of_a_subclass_that_know_no_adapters(monkeypatch):
    from omni_infer_amd.layers.deepseek_moe import DeepseekMoE

    class Block(DeepseekMoE):
        def _forward_norm_ops(self, hidden_states, attn_metadata):
            return hidden_states * 2

    b = _block(_Shared(), monkeypatch)
    b.__class__ = Block
    x = torch.randn(3, 8)
    assert torch.equal(b(x, None, None, 3)[0], x * 2)


def test_adapters_reach_a_shared_expert_that_has_room(monkeypatch):
    class Shared(_Shared):
        has_adapters = True

        def forward(self, x, adapters=None):
            return x + (1 if adapters is None else adapters)

    b = _block(Shared(), monkeypatch)
    x = torch.randn(3, 8)
    assert torch.equal(b(x, None, None, 3, adapters=5)[0], x + 5)
    assert torch.equal(b(x, None, None, 3)[0], x + 1)
