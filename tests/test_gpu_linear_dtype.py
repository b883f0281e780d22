"""A served model whose linear type or weights change: captured graphs and the prefix cache follow."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from aios_b200 import ImeCompletionEngine, ImeGenerationConfig, LLM
from aios_b200.kernel import ops
from aios_b200.models import init_synthetic_weights, shapes

pytestmark = pytest.mark.gpu

S10_L2 = dataclasses.replace(shapes.S10, num_layers=2)
S21_L4 = dataclasses.replace(shapes.S21, num_layers=4, attnres_num_blocks=2)


def _llm(config, **kwargs) -> tuple[LLM, ImeCompletionEngine]:
    llm = LLM(config=config, page_size=1, num_pages=2048, **{"seed": 0, **kwargs})
    return llm, ImeCompletionEngine(llm)


def _keystrokes(llm: LLM, engine: ImeCompletionEngine) -> list:
    """Short prefixes (graphs), one that extends the one before, and one that runs without a graph."""
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(10, llm.config.vocab_size, (90,), generator=g).tolist()
    out = []
    for n in (12, 12, 20, 90):
        result = engine.complete(llm.tokenizer.text_for(ids[:n]), ImeGenerationConfig(seed=4, max_new_tokens=6))
        out.append([(c.text, c.average_logprob) for c in result.raw_candidates])
    ops.check_status(llm.device)
    return out


def _fresh(config, **kwargs) -> list:
    return _keystrokes(*_llm(config, **kwargs))


@pytest.mark.parametrize("config", [S10_L2, S21_L4], ids=["S10", "S21"])
def test_a_switch_of_the_linear_type(cuda_device, config) -> None:
    want = {name: _fresh(config, linear_dtype=name) for name in ("bf16", "fp8")}
    assert want["bf16"] != want["fp8"]
    llm, engine = _llm(config)
    for name in ("bf16", "fp8", "fp8", "bf16", "fp8"):
        llm.model.set_linear_dtype(name)
        pool = torch.full((1 << 24,), 255, dtype=torch.uint8, device=cuda_device)  # takes memory that was let go
        assert _keystrokes(llm, engine) == want[name], name
        del pool


@pytest.mark.parametrize("name", ["bf16", "fp8"])
@pytest.mark.parametrize("config", [S10_L2, S21_L4], ids=["S10", "S21"])
def test_other_weights(cuda_device, config, name: str) -> None:
    want = {seed: _fresh(config, seed=seed, linear_dtype=name) for seed in (0, 1)}
    llm, engine = _llm(config, linear_dtype=name)
    for seed in (0, 1, 1, 0):
        init_synthetic_weights(llm.model, llm.device, seed=seed)
        assert llm.model.linear_dtype == name
        pool = torch.full((1 << 24,), 255, dtype=torch.uint8, device=cuda_device)
        assert _keystrokes(llm, engine) == want[seed], seed
        del pool


def test_the_persistent_step_goes_with_bf16(cuda_device) -> None:
    want = _fresh(S10_L2, linear_dtype="fp8")
    llm, engine = _llm(S10_L2)
    assert engine._runtime.use_persistent_step()
    _keystrokes(llm, engine)
    llm.model.set_linear_dtype("fp8")
    assert _keystrokes(llm, engine) == want
    assert engine._runtime._step_plan is None
    llm.model.set_linear_dtype("bf16")
    _keystrokes(llm, engine)
    assert engine._runtime._step_plan is not None


def test_a_copy_is_written_again_in_its_place(cuda_device) -> None:
    llm = LLM(config=S10_L2, seed=0, page_size=1, num_pages=64, linear_dtype="fp8")
    linear = llm.model.model.layers.op_list[0].self_attn.o_proj
    q, s = linear._fp8
    rows = ops.quantize_fp8(torch.randn(8, 768, device=cuda_device).to(torch.bfloat16))
    linear.forward_fp8(*rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear.forward_fp8(*rows)
    init_synthetic_weights(llm.model, llm.device, seed=1)
    assert linear._fp8[0].data_ptr() == q.data_ptr() and linear._fp8[1].data_ptr() == s.data_ptr()
    graph.replay()
    assert torch.equal(y, ops.linear_fp8(*rows, *ops.quantize_weight_fp8(linear.weight)))
    want = ops.quantize_weight_fp8(linear.weight)
    for wrong in (dict(out=q[:64]), dict(scale=s[:, :3]), dict(out=q.view(torch.uint8)), dict(scale=s.t())):
        with pytest.raises(ValueError, match="quantize_weight_fp8"):
            ops.quantize_weight_fp8(linear.weight, **wrong)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
