"""Draft batches of models on other roads than the fused bf16 one: an attention backend behind another, and 8-bit
linears."""

from __future__ import annotations

import math
import random

import pytest
import torch

from aios_b200.attention import B200AttentionBackend, HybridAttentionBackend
from aios_b200.core import Batch, Req
from aios_b200.kernel import ops
from tests import draft_reference as ref
from tests.test_gpu_draft_model import GREEDY, MODELS, IDS, Server, _prompts
from tests.test_gpu_fp8_model import _attnres_by_hand, _standard_by_hand

pytestmark = pytest.mark.gpu

TREES = [7, 13, 1, 40]
PROMPTS = [3, 40, 1, 150]


def _serve(cfg, linear_dtype: str, hybrid: bool = False) -> Server:
    prompts = _prompts(cfg, PROMPTS)
    s = Server(cfg, prompts)
    s.llm.model.set_linear_dtype(linear_dtype)
    if hybrid:
        model = s.llm.model
        backend = HybridAttentionBackend(B200AttentionBackend(cfg), B200AttentionBackend(cfg))
        model.attn_backend = model.model.attn_backend = s.llm.ctx.attn_backend = backend
        for layer in model.model.layers.op_list:
            layer.self_attn._attn_backend = backend
    s.prefill()
    return s


def _draft(s: Server, cfg) -> tuple[list[list[int]], torch.Tensor]:
    trees = ref.trees(TREES, "mixed", seed=5)
    rng = random.Random(2)
    drafted = [[t[-1]] + [rng.randrange(10, cfg.vocab_size) for _ in tree[1:]] for t, tree in zip(s.tokens, trees)]
    return trees, s.draft(trees, drafted)


@pytest.mark.parametrize("cfg", MODELS[:2], ids=IDS[:2])
def test_a_backend_behind_another(cuda_device, cfg) -> None:
    """With 8-bit linears the two roads run the same operators on the same values, so the logits are equal; with bf16
    ones the direct road folds its norms into the linears, and the log-probability of the likeliest token agrees within
    the parity tests' bar. Siblings share a position, so positions in order would be seen in both."""
    for linear_dtype in ("fp8", "bf16"):
        trees, direct = _draft(_serve(cfg, linear_dtype), cfg)
        s = _serve(cfg, linear_dtype, hybrid=True)
        _, behind = _draft(s, cfg)
        assert torch.equal(s.metadata.positions.cpu(), ref.tree_bits(trees, 2, s.cached)[1])
        if linear_dtype == "fp8":
            assert torch.equal(behind, direct)
        else:
            a, b = (torch.log_softmax(x.float(), dim=1) for x in (direct, behind))
            top = a.argmax(dim=1, keepdim=True)
            assert float((a.gather(1, top) - b.gather(1, top)).abs().max()) < 2e-2
        ops.check_status(cuda_device)


def test_a_draft_batch_holds_its_positions(cuda_device) -> None:
    """Also over positions that the caller had put there: the tree decides."""
    cfg = MODELS[0]
    s = _serve(cfg, "bf16")
    trees = [[-1, 0, 0, 1], [-1], [-1, 0], [-1]]
    reqs = [Req(input_ids=torch.zeros(c + len(t), dtype=torch.long), cached_len=c, output_len=4, uid=r,
                sampling_params=GREEDY, table_idx=r) for r, (t, c) in enumerate(zip(trees, s.cached))]
    for given in (None, torch.arange(8, dtype=torch.int32, device=s.llm.device)):
        b = Batch(reqs=reqs, phase="draft", trees=trees)
        b.out_loc = s.slots(8)
        if given is not None:
            b.positions = given
        s.llm.model.attn_backend.prepare_metadata(b)
        assert b.positions.tolist() == ref.tree_bits(trees, 1, s.cached)[1].tolist()


@pytest.mark.parametrize("cfg", MODELS, ids=IDS)
def test_8_bit_linears(cuda_device, cfg) -> None:
    """A draft forward's logits are those of its operators one by one in a layer's order, bit for bit, and as far from
    the bf16 model's as 8-bit prefills may be."""
    s = _serve(cfg, "fp8")
    caught = []

    def forward():
        out = LLMModel.forward(s.llm.model)
        batch = s.llm.ctx.batch
        caught.append((_attnres_by_hand if cfg is MODELS[2] else _standard_by_hand)(s.llm, batch))
        return out

    LLMModel = type(s.llm.model)
    s.llm.model.forward = forward
    _, got = _draft(s, cfg)
    assert torch.equal(got, caught[0])
    del s.llm.model.forward
    exact = _draft(_serve(cfg, "bf16"), cfg)[1].double()
    assert float((got.double() - exact).norm() / exact.norm()) < 0.051 * math.sqrt(7 * cfg.num_layers)
    ops.check_status(cuda_device)
