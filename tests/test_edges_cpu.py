"""Calls at the borders of the layer and of its operators that are refused, or decided on the host, checked
without a GPU."""

import pytest
import torch


def _layer(pkg, **kw):
    return pkg.SparseMoE(pkg.MoEConfig(**{**dict(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2), **kw}))


def test_logit_bias_has_one_entry_per_expert(moe_pkg):
    layer = _layer(moe_pkg)
    cpu = torch.device("cpu")
    assert layer._logit_bias(cpu, 8) is None
    for n in (7, 9):
        layer.router_logit_bias = torch.zeros(n)
        with pytest.raises(ValueError, match="router_logit_bias"):
            layer._logit_bias(cpu, 8)
    layer.router_logit_bias = torch.arange(8, dtype=torch.bfloat16)
    assert torch.equal(layer._logit_bias(cpu, 8), torch.arange(8, dtype=torch.float32))
