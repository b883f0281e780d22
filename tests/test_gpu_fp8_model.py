"""Models served with 8-bit linears (``LLM(linear_dtype="fp8")``).

* wiring: the logits equal, bit for bit, those of the same operators called one by one in a
  decoder layer's order;
* size of the error, in the 2-norm against the bf16 model's logits. Quantising a value is off
  by a uniform error of at most 2^-4 of it: at most 2^-4 / sqrt(3) = 3.6% root mean square. A
  linear whose rows and weight are both quantised is off by at most sqrt(2) * 3.6% = 5.1% of
  its output. Errors of different linears are independent, so their variances add on the way
  to the logits, norms pass relative errors on unchanged, and the residual stream's sum is off
  by no more than its worst term. In units of 5.1% squared a layer brings 1 for qkv, 1 for o,
  4 for gate/up (SwiGLU multiplies two of its outputs, and silu's relative slope is below 1.3
  on average) and 1 for down: sqrt(7 * layers) * 5.1%;
* the engine on top: captured steps, scoring in both modes and generation.
"""

from __future__ import annotations

import dataclasses
import math

import pytest
import torch

from aios_b200 import ImeCompletionEngine, ImeGenerationConfig, LLM, SamplingParams
from aios_b200 import _lib
from aios_b200.core import Batch, Req
from aios_b200.kernel import ops
from aios_b200.models import shapes
from aios_b200.models.minimind_ime import mix_and_norm

pytestmark = pytest.mark.gpu

S10_L2 = dataclasses.replace(shapes.S10, num_layers=2)
S06_L2 = dataclasses.replace(shapes.S06, num_layers=2)
S21_L4 = dataclasses.replace(shapes.S21, num_layers=4, attnres_num_blocks=2)


def _prefill_batch(llm: LLM, lengths: list[int], seed: int = 3) -> Batch:
    g = torch.Generator().manual_seed(seed)
    dev = llm.device
    reqs, slots, pos, at = [], [], [], 0
    llm.ctx.page_table = torch.zeros((len(lengths), max(lengths)), dtype=torch.int32, device=dev)
    for i, n in enumerate(lengths):
        reqs.append(Req(input_ids=torch.empty(n, dtype=torch.long), cached_len=0, output_len=1, uid=i,
                        sampling_params=SamplingParams(max_tokens=1), table_idx=i))
        llm.ctx.page_table[i, :n] = torch.arange(at, at + n, dtype=torch.int32, device=dev)
        slots += range(at, at + n)
        pos += range(n)
        at += n
    batch = Batch(reqs=reqs, phase="prefill", return_all_logits=True)
    batch.input_ids = torch.randint(0, llm.config.vocab_size, (at,), generator=g, dtype=torch.int32).to(dev)
    batch.positions = torch.tensor(pos, dtype=torch.int32, device=dev)
    batch.out_loc = torch.tensor(slots, dtype=torch.int32, device=dev)
    llm.model.attn_backend.prepare_metadata(batch)
    return batch


def _logits(llm: LLM, batch: Batch) -> torch.Tensor:
    with llm.ctx.forward_batch(batch):
        out = llm.model.forward()
    torch.cuda.synchronize()
    ops.check_status(llm.device)
    return out


def _standard_by_hand(llm: LLM, batch: Batch) -> torch.Tensor:
    m = llm.model.model
    eps = llm.config.rms_norm_eps
    x = ops.embedding(batch.input_ids, m.embed_tokens.weight)
    residual = None
    for layer in m.layers.op_list:
        at, mlp = layer.self_attn, layer.mlp
        w = [ops.quantize_weight_fp8(t.weight) for t in (at.qkv_proj, at.o_proj, mlp.gate_up_proj, mlp.down_proj)]
        if residual is None:
            rows, residual = ops.rmsnorm_fp8(x, layer.input_layernorm.weight, eps), x
        else:
            rows = ops.fused_add_rmsnorm_fp8(x, residual, layer.input_layernorm.weight, eps)
        a = at.attend_qkv(ops.linear_fp8(*rows, *w[0]), m._rotary_emb, llm.ctx.kv_cache, batch)
        x = ops.linear_fp8(*ops.quantize_fp8(a), *w[1])
        rows = ops.fused_add_rmsnorm_fp8(x, residual, layer.post_attention_layernorm.weight, eps)
        x = ops.linear_fp8(*ops.silu_and_mul_fp8(ops.linear_fp8(*rows, *w[2])), *w[3])
    ops.fused_add_rmsnorm(x, residual, m.norm.weight, eps)
    return ops.linear(x, llm.model.lm_head._w())


def _attnres_by_hand(llm: LLM, batch: Batch) -> torch.Tensor:
    m, cfg = llm.model.model, llm.config
    per = cfg.layers_per_attnres_block
    bank = ops.embedding(batch.input_ids, m.embed_tokens.weight).unsqueeze(0)
    mixed = torch.empty_like(bank[0])
    for block in range(cfg.attnres_num_blocks):
        partial = None
        for layer in m.layers.op_list[block * per : (block + 1) * per]:
            at, mlp = layer.self_attn, layer.mlp
            w = [ops.quantize_weight_fp8(t.weight) for t in (at.qkv_proj, at.o_proj, mlp.gate_up_proj, mlp.down_proj)]
            h = mix_and_norm(layer.attn_res_mixer, layer.input_layernorm, bank, partial, mixed)
            a = at.attend_qkv(ops.linear_fp8(*ops.quantize_fp8(h), *w[0]), m._rotary_emb, llm.ctx.kv_cache, batch)
            rows = ops.quantize_fp8(a)
            if partial is None:
                partial = ops.linear_fp8(*rows, *w[1])
            else:
                partial = ops.linear_fp8(*rows, *w[1], epilogue=_lib.EPI_ADD, residual=partial)
            h = mix_and_norm(layer.mlp_res_mixer, layer.post_attention_layernorm, bank, partial, mixed)
            act = ops.silu_and_mul_fp8(ops.linear_fp8(*ops.quantize_fp8(h), *w[2]))
            partial = ops.linear_fp8(*act, *w[3], epilogue=_lib.EPI_ADD, residual=partial)
        bank = torch.cat((bank, partial.unsqueeze(0))).contiguous()
    hidden = m.final_attn_res_mixer.forward(bank)
    return ops.linear(ops.rmsnorm(hidden, m.norm.weight, cfg.rms_norm_eps), llm.model.lm_head._w())


@pytest.mark.parametrize("lengths", [[1], [13], [5, 70, 1, 40], [300, 200]])
@pytest.mark.parametrize("config", [S10_L2, S06_L2, S21_L4], ids=["S10", "S06", "S21"])
def test_logits_are_the_operators_in_order(cuda_device, config, lengths) -> None:
    llm = LLM(config=config, seed=0, page_size=1, num_pages=1024, linear_dtype="fp8")
    assert llm.model.linear_dtype == "fp8"
    batch = _prefill_batch(llm, lengths)
    got = _logits(llm, batch)
    with llm.ctx.forward_batch(batch):
        want = (_attnres_by_hand if config is S21_L4 else _standard_by_hand)(llm, batch)
    assert torch.equal(got, want)
    llm.model.set_linear_dtype("bf16")
    exact = _logits(llm, batch).double()
    assert float((got.double() - exact).norm() / exact.norm()) < 0.051 * math.sqrt(7 * config.num_layers)
    llm.model.set_linear_dtype("fp8")
    assert torch.equal(_logits(llm, batch), got)


@pytest.mark.parametrize("config", [S10_L2, S21_L4], ids=["S10", "S21"])
def test_engine_on_8_bit_linears(cuda_device, config) -> None:
    """Keystrokes through prefill and step graphs, twice the same; scores of both modes agree
    (their batches differ, so a value next to a rounding border may step by 2^-4 of itself:
    averages within 0.1 in log-probability)."""
    llm = LLM(config=config, seed=0, page_size=1, num_pages=2048, linear_dtype="fp8")
    engine = ImeCompletionEngine(llm)
    g = torch.Generator().manual_seed(5)
    text = llm.tokenizer.text_for(torch.randint(10, config.vocab_size, (12,), generator=g).tolist())
    runs = []
    for _ in range(2):
        engine.reset_prefix_cache()
        result = engine.complete(text, ImeGenerationConfig(seed=4, max_new_tokens=8))
        runs.append([(c.text, c.average_logprob) for c in result.raw_candidates])
    assert len(runs[0]) >= 8 and runs[0] == runs[1]
    cands = [llm.tokenizer.text_for(torch.randint(10, config.vocab_size, (n,), generator=g).tolist())
             for n in (1, 4, 9)]
    stable = engine.score_candidates(text, cands, mode="stable")
    shared = engine.score_candidates(text, cands, mode="shared_decode")
    a = {c.text: c.average_logprob for c in stable.candidates}
    b = {c.text: c.average_logprob for c in shared.candidates}
    assert set(a) == set(cands) == set(b)
    for c in cands:
        assert abs(a[c] - b[c]) < 0.1
    ops.check_status(llm.device)


def test_generate_on_8_bit_linears(cuda_device) -> None:
    llm = LLM(config=S10_L2, seed=0, page_size=1, num_pages=2048, linear_dtype="fp8")
    prompts = [[5, 9, 200, 31], list(range(20, 120)), [7]]
    out = llm.generate(prompts, SamplingParams(max_tokens=6, ignore_eos=True))
    assert [len(o["token_ids"]) for o in out] == [6, 6, 6]
    assert out == llm.generate(prompts, SamplingParams(max_tokens=6, ignore_eos=True))


def test_linear_dtype_is_checked(cuda_device) -> None:
    with pytest.raises(ValueError, match="linear_dtype must be"):
        LLM(config=S10_L2, seed=0, page_size=1, num_pages=64, linear_dtype="int8")
    llm = LLM(config=S10_L2, seed=0, page_size=1, num_pages=64)
    assert llm.model.linear_dtype == "bf16"
    layer = llm.model.model.layers.op_list[0]
    with pytest.raises(RuntimeError, match="quantize_fp8"):
        layer.self_attn.o_proj.forward_fp8(*ops.quantize_fp8(torch.zeros(1, 768, dtype=torch.bfloat16, device="cuda")))
