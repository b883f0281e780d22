"""Drafted trees through a model, as they are used: a draft batch's forward (positions and bits from the
parents, prologue, tree attention in every layer), the verification, and the page table's entries kept in
the verification's order.
"""

from __future__ import annotations

import dataclasses
import random

import pytest
import torch

from aios_b200 import LLM
from aios_b200.core import Batch, Req, SamplingParams
from aios_b200.engine import Sampler
from aios_b200.models import shapes
from oracle.model import Request
from tests import draft_reference as ref
from tests.test_gpu_generate import _oracle

pytestmark = pytest.mark.gpu

MODELS = [dataclasses.replace(shapes.S10, num_layers=2), dataclasses.replace(shapes.S06, num_layers=2),
          dataclasses.replace(shapes.S21, num_layers=4, attnres_num_blocks=2)]
IDS = ["s10_l2", "s06_l2", "s21_l4"]
GREEDY = SamplingParams(temperature=0.0, max_tokens=64)


class Server:
    """Requests with page-table rows of their own; slots are taken in order from the pool."""

    def __init__(self, cfg, prompts: list[list[int]], page_size: int = 1):
        self.llm = LLM(config=cfg, seed=0, page_size=page_size, num_pages=2048 // page_size)
        self.table = torch.zeros((len(prompts), 300), dtype=torch.int32, device=self.llm.device)
        self.llm.ctx.page_table = self.table
        self.next_slot = 5
        self.tokens = [list(p) for p in prompts]  # known tokens: all but the last are in the cache
        self.cached = [0] * len(prompts)

    def slots(self, n: int) -> torch.Tensor:
        out = torch.arange(self.next_slot, self.next_slot + n, dtype=torch.int32, device=self.llm.device)
        self.next_slot += n
        return out

    def forward(self, phase: str, rows: list[int], ids: list[list[int]], cached: list[int], **kw) -> torch.Tensor:
        reqs, out_loc, positions = [], [], []
        for r, new, c in zip(rows, ids, cached):
            req = Req(input_ids=torch.zeros(c + len(new), dtype=torch.long), cached_len=c, output_len=64, uid=r,
                      sampling_params=GREEDY, table_idx=r)
            slots = self.slots(len(new))
            self.table[r, c : c + len(new)] = slots
            reqs.append(req)
            out_loc.append(slots)
            positions += range(c, c + len(new))
        b = Batch(reqs=reqs, phase=phase, **kw)
        b.input_ids = torch.tensor([t for new in ids for t in new], device=self.llm.device)
        if phase == "prefill":
            b.positions = torch.tensor(positions, dtype=torch.int32, device=self.llm.device)
        b.out_loc = torch.cat(out_loc)
        self.llm.model.attn_backend.prepare_metadata(b)
        with torch.no_grad(), self.llm.ctx.forward_batch(b):
            logits = self.llm.model.forward()
        self.metadata = b.attn_metadata
        return logits

    def prefill(self) -> None:
        """All known tokens but the last into the cache."""
        rows = list(range(len(self.tokens)))
        self.forward("prefill", rows, [t[:-1] for t in self.tokens], self.cached)
        self.cached = [len(t) - 1 for t in self.tokens]

    def draft(self, trees: list[list[int]], drafted: list[list[int]]) -> torch.Tensor:
        """One draft forward; drafted[r][0] is the request's last known token."""
        return self.forward("draft", list(range(len(trees))), drafted, self.cached, trees=trees)

    def keep(self, trees, drafted, accepted, order, token) -> None:
        at = 0
        for r, tree in enumerate(trees):
            n, c, stay = len(tree), self.cached[r], int(accepted[r]) + 1
            path = order[at : at + n].long()
            self.table[r, c : c + n] = self.table[r, c : c + n][path]
            nodes = path[:stay].tolist()
            assert self.tokens[r][-1] == drafted[r][nodes[0]]
            self.tokens[r] += [drafted[r][i] for i in nodes[1:]] + [int(token[r])]
            self.cached[r] = c + stay
            at += n


def _prompts(cfg, lengths, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [[1] + torch.randint(10, cfg.vocab_size, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("cfg", MODELS, ids=IDS)
@pytest.mark.parametrize("page_size", [1, 16])
def test_a_nodes_logits_are_those_of_its_path(cfg, page_size) -> None:
    """Every node against a prefill of the prompt and the node's ancestors: the same model by other kernels, so
    within the bar of the parity tests (2e-2 on the log-probability of the likeliest token)."""
    prompts = _prompts(cfg, [3, 40, 1, 150])
    s = Server(cfg, prompts, page_size)
    s.prefill()
    trees = ref.trees([7, 13, 1, 40], "mixed", seed=5)
    rng = random.Random(2)
    drafted = [[p[-1]] + [rng.randrange(10, cfg.vocab_size) for _ in t[1:]] for p, t in zip(prompts, trees)]
    got = torch.log_softmax(s.draft(trees, drafted).float(), dim=1)
    assert got.shape[0] == sum(len(t) for t in trees)
    mask, positions = ref.tree_bits(trees, 2, s.cached)
    assert torch.equal(s.metadata.positions.cpu(), positions) and torch.equal(s.metadata.tree_mask.cpu(), mask)
    table, slot = s.table.clone(), s.next_slot
    at = 0
    for r, tree in enumerate(trees):
        for i in range(0, len(tree), 3):
            path, j = [], i
            while j >= 0:
                path.append(drafted[r][j])
                j = tree[j]
            s.next_slot = slot
            row = s.forward("prefill", [r], [prompts[r][:-1] + path[::-1]], [0])
            want = torch.log_softmax(row[0].float(), dim=0)
            top = int(want.argmax())
            assert abs(float(got[at + i, top] - want[top])) < 2e-2, (r, i)
            s.table.copy_(table)
        at += len(tree)


LOGPROB_BAR = 2e-2  # of a log-probability against the oracle's, as in the parity tests


def _flips(oracle, prompt: list[int], generated: list[int]) -> int:
    """The generated tokens that are not the oracle's argmax, teacher-forced. Where two logits are each off by at
    most the bar, they can change places only if they lie within twice the bar."""
    ids = prompt + generated
    n = len(ids)
    flips = 0
    for end in range(len(prompt), n):
        row = oracle.forward([Request(ids=ids[:end], positions=list(range(end)), new_slots=list(range(end)),
                                      key_slots=list(range(end)))])[-1].float()
        gap = float(row.max() - row[ids[end]])
        assert gap <= 2 * LOGPROB_BAR, (end, gap)
        flips += gap > 0
    return flips


@pytest.mark.parametrize("cfg", MODELS, ids=IDS)
def test_greedy_drafting_gives_the_greedy_tokens(cfg) -> None:
    """Trees whose proposals are partly the model's own continuation (from a first, sequential run): the tokens that
    drafting yields, replayed on the oracle, are its argmax but for near-ties."""
    prompts = _prompts(cfg, [5, 33, 2])
    params = SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True)
    llm = LLM(config=cfg, seed=0, page_size=1, num_pages=512)
    known = [r["token_ids"] for r in llm.generate(prompts, params)]
    s = Server(cfg, prompts)
    s.prefill()
    sampler, rng = Sampler(GREEDY), random.Random(7)
    steps, kept = 0, 0
    while min(len(t) - len(p) for t, p in zip(s.tokens, prompts)) < 16:
        trees, drafted = [], []
        for t, p, k in zip(s.tokens, prompts, known):
            done = len(t) - len(p)
            right = k[done : done + 3] if t[len(p) :] == k[:done] else []
            # a chain of right tokens, wrong siblings hung before and below them
            tree, ids, last = [-1], [t[-1]], 0
            for x in right:
                for _ in range(rng.randrange(3)):
                    tree.append(last)
                    ids.append((x + rng.randrange(1, 50)) % cfg.vocab_size)
                tree.append(last)
                ids.append(x)
                last = len(tree) - 1
                tree.append(last)
                ids.append(rng.randrange(10, cfg.vocab_size))
            trees.append(tree)
            drafted.append(ids)
        logits = s.draft(trees, drafted)
        md = s.metadata
        flat = torch.tensor([x for d in drafted for x in d], device=logits.device)
        accepted, token, order = sampler.verify(logits, flat, md.parents, md.tree_start)
        s.keep(trees, drafted, accepted.tolist(), order, token.tolist())
        steps += 1
        kept += int(accepted.sum())
    oracle = _oracle(cfg, 1024)
    flips = sum(_flips(oracle, p, t[len(p) : len(p) + 16]) for p, t in zip(prompts, s.tokens))
    assert flips <= 4
    assert kept > steps  # drafting did carry several tokens a forward


def test_sampled_drafting_on_the_sampler(cuda_device) -> None:
    """Sampler.verify: its own draws from a generator are those of the operator with the same numbers; filters are
    refused; equal logits by any road."""
    from aios_b200.kernel import ops

    g = torch.Generator().manual_seed(1)
    trees = ref.trees([9, 4], "mixed", 1)
    flat = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 9, 13], dtype=torch.int32, device="cuda")
    logits = (2 * torch.randn(13, 700, generator=g)).to(torch.bfloat16).cuda()
    drafts = torch.randint(0, 700, (13,), generator=g).cuda()
    probs = torch.softmax(logits.float() + 0.5, dim=1)
    sampler = Sampler(SamplingParams(temperature=0.7))
    gen = torch.Generator(device="cuda").manual_seed(11)
    got = sampler.verify(logits, drafts, flat, start, draft_probs=probs, generator=gen)
    gen.manual_seed(11)
    u, v = torch.rand(13, generator=gen, device="cuda"), torch.rand(2, generator=gen, device="cuda")
    want = ops.verify_draft(logits, drafts, flat, start, u, v, temperature=0.7, draft_probs=probs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = sampler.verify(logits, drafts, flat, start, draft_probs=probs, accept_uniforms=u, sample_uniforms=v)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    with pytest.raises(ValueError, match="exclusive"):
        sampler.verify(logits, drafts, flat, start, generator=gen, accept_uniforms=u)
    for params in (SamplingParams(temperature=0.7, top_k=20), SamplingParams(temperature=0.7, top_p=0.9)):
        with pytest.raises(ValueError, match="mask the logits"):
            Sampler(params).verify(logits, drafts, flat, start)


def test_a_draft_batch_refuses(cuda_device) -> None:
    cfg = MODELS[0]
    s = Server(cfg, _prompts(cfg, [3]))
    s.prefill()
    with pytest.raises(ValueError, match="one tree"):
        s.forward("draft", [0], [[5, 6]], s.cached)
    with pytest.raises(ValueError, match="one slot"):
        s.forward("draft", [0], [[5, 6]], s.cached, trees=[[-1]])
    with pytest.raises(ValueError, match="before their children"):
        s.forward("draft", [0], [[5, 6]], s.cached, trees=[[-1, 1]])
    with pytest.raises(ValueError, match="nodes"):
        s.forward("draft", [0], [[]], s.cached, trees=[[]])
