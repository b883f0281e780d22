"""The model's key for captured graphs and for cached K/V (no GPU)."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from aios_b200.models import shapes
from aios_b200.models.minimind_ime import MiniMindIMEForCausalLM
from aios_b200.models.weight import init_synthetic_weights

S06_L1 = dataclasses.replace(shapes.S06, num_layers=1)
S21_L2 = dataclasses.replace(shapes.S21, num_layers=2, attnres_num_blocks=1)


@pytest.mark.parametrize("config", [S06_L1, S21_L2], ids=["standard", "attnres"])
def test_graph_key_follows_weights_and_linear_type(config) -> None:
    with torch.device("meta"):
        model = MiniMindIMEForCausalLM(config)
    keys = [model.graph_key]
    for seed in (0, 0):
        init_synthetic_weights(model, torch.device("cpu"), seed=seed)
        keys.append(model.graph_key)
    model.set_linear_dtype("bf16")  # no change
    assert model.graph_key == keys[-1]
    model.model._fp8_linears = True
    keys.append(model.graph_key)
    assert len(set(keys)) == 4
    init_synthetic_weights(model, torch.device("cpu"), seed=1)  # 8-bit copies are built on the GPU
    assert model.linear_dtype == "fp8" and model.graph_key not in keys


def test_a_copy_of_replaced_weights_is_not_used() -> None:
    with torch.device("meta"):
        model = MiniMindIMEForCausalLM(S06_L1)
    init_synthetic_weights(model, torch.device("cpu"))
    linear = model.model.layers.op_list[0].self_attn.o_proj
    linear._fp8, linear._fp8_stale = (torch.zeros(1), torch.zeros(1)), False
    init_synthetic_weights(model, torch.device("cpu"), seed=1)
    with pytest.raises(RuntimeError, match="quantize_fp8"):
        linear.forward_fp8(torch.zeros(1, 768), torch.zeros(1, 6))
    assert linear._fp8 is not None  # kept: a captured graph may read it
