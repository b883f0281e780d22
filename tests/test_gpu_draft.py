"""draft_tree and verify_draft against plain restatements in fp64: whole numbers, so equal."""

from __future__ import annotations

import pytest
import torch

from aios_b200 import _lib
from aios_b200.kernel import ops
from tests import draft_reference as ref

pytestmark = pytest.mark.gpu


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _flat(parents: list[list[int]]) -> torch.Tensor:
    return _i32([p for ps in parents for p in ps])


# ---- draft_tree --------------------------------------------------------------
@pytest.mark.parametrize("kind", ["chain", "star", "mixed"])
@pytest.mark.parametrize("sizes", [[1], [8], [0, 3, 0, 33, 1, 0], [32, 64, 31], [200, 256], [1024, 700]])
@pytest.mark.parametrize("with_cached", [True, False])
def test_draft_tree(cuda_device, kind: str, sizes: list[int], with_cached: bool) -> None:
    parents = ref.trees(sizes, kind)
    most = max(sizes)
    cached = [17 * r + 5 for r in range(len(sizes))] if with_cached else None
    want_mask, want_pos = ref.tree_bits(parents, (most + 31) // 32, cached)
    tokens = sum(sizes)
    flat = torch.cat([_flat(parents), _i32([-7] * 3)])  # rows behind the last tree
    mask = torch.full((tokens + 3, (most + 31) // 32), -9, dtype=torch.int32, device="cuda")
    pos = torch.full((tokens + 3,), -9, dtype=torch.int32, device="cuda")
    got = ops.draft_tree(flat, _i32(ref.starts(sizes)), max_nodes=most, cached_lens=_i32(cached) if cached else None,
                         mask=mask, positions=pos)
    assert got[0] is mask and got[1] is pos
    assert torch.equal(mask[:tokens].cpu(), want_mask) and torch.equal(pos[:tokens].cpu(), want_pos)
    assert (mask[tokens:] == -9).all() and (pos[tokens:] == -9).all()
    ops.check_status(cuda_device)


def test_a_forest_is_a_tree_with_several_roots(cuda_device) -> None:
    parents = [[-1, -1, 0, 1, 3, -1]]
    want = ref.tree_bits(parents, 1)
    mask, pos = ops.draft_tree(_flat(parents), _i32([0, 6]), max_nodes=6)
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(pos.cpu(), want[1])


@pytest.mark.parametrize("parents,starts,most", [
    ([-1, 1, 0], [0, 3], 3),  # its own parent
    ([-1, 2, 0], [0, 3], 3),  # a later one
    ([-1, 0, -2], [0, 3], 3),
    ([-1, 0, 1], [0, 4], 3),  # past the arrays
    ([-1, 0, 1], [2, 1], 3),  # descending
    ([-1, 0, 1], [-1, 3], 3),
    ([i - 1 for i in range(40)], [0, 40], 32),  # more nodes than words
    ([i - 1 for i in range(1100)], [0, 1100], 1024),
])
def test_bad_trees_are_reported(cuda_device, parents, starts, most) -> None:
    ops.draft_tree(_i32(parents), _i32(starts), max_nodes=most)
    with pytest.raises(RuntimeError, match="tree"):
        ops.check_status(cuda_device)


def test_draft_tree_refuses(cuda_device) -> None:
    p, s = _i32([-1, 0]), _i32([0, 2])
    for bad in (lambda: ops.draft_tree(p.long(), s, max_nodes=2), lambda: ops.draft_tree(p[None], s, max_nodes=2),
                lambda: ops.draft_tree(p, s.long(), max_nodes=2), lambda: ops.draft_tree(p, s, max_nodes=0),
                lambda: ops.draft_tree(p, s, max_nodes=1025), lambda: ops.draft_tree(p, s.cpu(), max_nodes=2),
                lambda: ops.draft_tree(p, s, max_nodes=2, cached_lens=p),
                lambda: ops.draft_tree(p, s, max_nodes=2, positions=p.long()),
                lambda: ops.draft_tree(p, s, max_nodes=2, mask=p)):
        with pytest.raises(ValueError, match="draft_tree"):
            bad()
    empty = ops.draft_tree(p[:0], s[:1], max_nodes=2)
    assert empty[0].shape == (0, 1) and empty[1].shape == (0,)


# ---- verify_draft ------------------------------------------------------------
def _case(sizes, vocab, kind="mixed", dtype=torch.bfloat16, probs=False, seed=0, spread=2.5, distinct=True, extra=0):
    g = torch.Generator().manual_seed(seed)
    parents = ref.trees(sizes, kind, seed)
    tokens = sum(sizes)
    logits = (spread * torch.randn(tokens + extra, vocab, generator=g)).to(dtype)
    near = logits.float() + 0.7 * torch.randn(tokens + extra, vocab, generator=g)
    q = torch.softmax(near, dim=1) if probs else None
    drafts = torch.zeros(tokens + extra, dtype=torch.int64)
    at = 0
    for ps in parents:
        for i in range(1, len(ps)):
            siblings = sum(1 for j in range(1, i) if ps[j] == ps[i])
            row = at + ps[i]
            if probs:
                drafts[at + i] = torch.multinomial(q[row], 1, generator=g)[0]
            elif distinct:
                drafts[at + i] = torch.topk(near[row], min(vocab, siblings + 1)).indices[-1]
            else:
                drafts[at + i] = torch.randint(0, vocab, (1,), generator=g)[0]
        at += len(ps)
    accept = torch.rand(tokens + extra, generator=g)
    sample = torch.rand(len(sizes), generator=g)
    return parents, logits, drafts, accept, sample, q


def _run(case, sizes, **kwargs):
    parents, logits, drafts, accept, sample, q = case
    pad = logits.shape[0] - sum(sizes)
    flat = torch.cat([_flat(parents), _i32([-5] * pad)]) if pad else _flat(parents)
    got = ops.verify_draft(logits.cuda(), drafts.cuda(), flat, _i32(ref.starts(sizes)), accept.cuda(), sample.cuda(),
                           draft_probs=None if q is None else q.cuda(), **kwargs)
    return [t.tolist() for t in got]


SIZES = [[1], [5], [2, 0, 9, 1], [26, 13, 33, 1, 17], [0, 0], [70, 100]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 6401, 32768])
@pytest.mark.parametrize("mode", ["greedy", "plain", "probs", "chain"])
def test_verify(cuda_device, sizes, vocab: int, mode: str) -> None:
    for seed in range(3):
        kind = "chain" if mode == "chain" else "mixed"
        case = _case(sizes, vocab, kind, torch.float32 if seed == 1 else torch.bfloat16, mode in ("probs", "chain"),
                     seed, spread=(2.5, 0.3, 8.0)[seed])
        kw = {"greedy": True} if mode == "greedy" else {"temperature": (1.0, 0.7, 1.3)[seed]}
        want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5], **kw)
        assert _run(case, sizes, **kw) == [list(w) for w in want]
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [50021, 131072, 151111, 160001, 262137, 262144])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_vocabularies(cuda_device, vocab: int, probs: bool) -> None:
    sizes = [12, 7, 1]
    case = _case(sizes, vocab, probs=probs, seed=vocab)
    want = ref.verify(case[1], case[2], case[0], case[3], case[4], temperature=0.8, probs=case[5])
    assert _run(case, sizes, temperature=0.8) == [list(w) for w in want]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off", range(8))
@pytest.mark.parametrize("mode", ["greedy", "plain", "probs"])
def test_rows_anywhere_on_16_bytes(cuda_device, dtype, off: int, mode: str) -> None:
    """Every place of a row and of its probabilities, NaN around both."""
    for vocab in (1, 6, 255, 1030):
        sizes = [3, 6]
        case = _case(sizes, vocab, dtype=dtype, probs=mode == "probs", seed=off)
        parents, logits, drafts, accept, sample, q = case
        kw = {"greedy": True} if mode == "greedy" else {}
        want = ref.verify(logits, drafts, parents, accept, sample, probs=q, **kw)
        for stride in (vocab + 16, vocab + 21):
            wide = torch.full((9, stride), float("nan"), dtype=dtype, device="cuda")
            wide[:, off : off + vocab] = logits.cuda()
            wide_q = torch.full((9, stride + 2), float("nan"), device="cuda")
            at = (3 * off + 1) % 8
            if q is not None:
                wide_q[:, at : at + vocab] = q.cuda()
            got = ops.verify_draft(wide[:, off : off + vocab], drafts.cuda(), _flat(parents), _i32([0, 3, 9]),
                                   accept.cuda(), sample.cuda(),
                                   draft_probs=wide_q[:, at : at + vocab] if q is not None else None, **kw)
            assert [t.tolist() for t in got] == [list(w) for w in want]
    ops.check_status(cuda_device)


@pytest.mark.parametrize("kind", ["star", "chain", "mixed"])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_trees(cuda_device, kind: str, probs: bool) -> None:
    """More children than a warp has lanes, the longest path, as many nodes as a tree may have."""
    sizes = [1024, 70]
    case = _case(sizes, 90, kind, torch.float32, probs, seed=4, spread=0.2)
    case[3].mul_(0.2 if kind == "chain" else 1.0)
    if kind == "star":
        case[3][1:60] = 0.9999
    want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5])
    assert _run(case, sizes) == [list(w) for w in want]


@pytest.mark.parametrize("requests", [1, 8, 37, 150, 400])
def test_verify_many_requests(cuda_device, requests: int) -> None:
    sizes = [1 + i % 4 for i in range(requests)]
    for probs in (False, True):
        case = _case(sizes, 517, probs=probs, seed=requests)
        want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5])
        assert _run(case, sizes) == [list(w) for w in want]


def test_the_ends_of_the_uniforms(cuda_device) -> None:
    sizes = [9, 9]
    for u in (0.0, 1.0 - 2.0**-24):
        for probs in (False, True):
            case = _case(sizes, 777, probs=probs, seed=3)
            case[3].fill_(u)
            case[4].fill_(u)
            want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5])
            assert _run(case, sizes) == [list(w) for w in want]


def test_equal_proposals_and_equal_logits(cuda_device) -> None:
    """The same token twice below one node (rejected, it is gone), and ties of the argmax."""
    sizes = [6]
    case = _case(sizes, 64, "star", seed=1)
    case[2][1:] = 5
    case[3].fill_(0.999)
    want = ref.verify(case[1], case[2], case[0], case[3], case[4])
    assert _run(case, sizes) == [list(w) for w in want]
    case[1].zero_()
    case[2][1:] = torch.tensor([3, 1, 0, 0, 2])
    assert _run(case, sizes, greedy=True) == [[1], [0], [0, 3, 1, 2, 4, 5]]


def test_a_draft_equal_to_the_target_leaves_nothing(cuda_device) -> None:
    """q = p: a rejection (u over 1 forces one) leaves max(p - q, 0) = 0 everywhere but for rounding;
    where it is 0 exactly the distribution stays."""
    logits = torch.zeros(2, 4, dtype=torch.bfloat16)
    q = torch.full((2, 4), 0.25)
    parents = [[-1, 0]]
    args = (logits.cuda(), torch.tensor([0, 2]).cuda(), _flat(parents), _i32([0, 2]), torch.tensor([0.0, 1.5]).cuda(),
            torch.tensor([0.6]).cuda())
    accepted, token, order = ops.verify_draft(*args, draft_probs=q.cuda())
    assert accepted.tolist() == [0] and token.tolist() == [2] and order.tolist() == [0, 1]


@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 0.02, 30.0, 1e6])
@pytest.mark.parametrize("spread", [1e-3, 3.0, 3e4])
def test_temperatures(cuda_device, temperature: float, spread: float) -> None:
    sizes = [9, 4]
    for probs in (False, True):
        case = _case(sizes, 1200, probs=probs, seed=8, dtype=torch.float32, spread=spread)
        case[1][:, 1000:1100] = -float("inf")
        want = ref.verify(case[1], case[2], case[0], case[3], case[4], temperature=temperature, probs=case[5])
        assert _run(case, sizes, temperature=temperature) == [list(w) for w in want]
    ops.check_status(cuda_device)


def test_masked_logits(cuda_device) -> None:
    """A sampler's filter: -inf takes a token out, as a proposal and as the next token."""
    sizes = [9, 4]
    for probs in (False, True):
        case = _case(sizes, 300, probs=probs, seed=8)
        case[1][:, 50:] = -float("inf")
        case[1][0, 7] = -float("inf")
        want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5])
        got = _run(case, sizes)
        assert got == [list(w) for w in want] and all(t < 50 for t in got[1])
    ops.check_status(cuda_device)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("greedy", [False, True])
def test_rows_without_a_distribution(cuda_device, value: float, greedy: bool) -> None:
    case = _case([1, 1, 1], 1500, seed=2)
    if value == -float("inf"):
        case[1][1] = value
    else:
        case[1][1, 1499] = value
    kw = {"greedy": greedy}
    want = ref.verify(case[1], case[2], case[0], case[3], case[4], **kw)
    got = _run(case, [1, 1, 1], **kw)
    assert got == [list(w) for w in want]
    if greedy and value == float("inf"):
        assert got[1][1] == 1499
        ops.check_status(cuda_device)
    else:
        assert got[1][1] == -1
        with pytest.raises(RuntimeError, match="no token"):
            ops.check_status(cuda_device)


def test_draft_tokens_outside_the_vocabulary(cuda_device) -> None:
    for mode in ({"greedy": True}, {}):
        for probs in (False, True):
            if probs and mode:
                continue
            case = _case([5], 200, "star", probs=probs, seed=4)
            case[2][1], case[2][2] = 200, -1
            want = ref.verify(case[1], case[2], case[0], case[3], case[4], probs=case[5], **mode)
            assert _run(case, [5], **mode) == [list(w) for w in want]
            with pytest.raises(RuntimeError, match="vocabulary"):
                ops.check_status(cuda_device)


def test_rows_behind_the_last_tree_and_strides(cuda_device) -> None:
    sizes = [5, 3]
    case = _case(sizes, 333, probs=True, seed=6, extra=4)
    parents, logits, drafts, accept, sample, q = case
    want = ref.verify(logits, drafts, parents, accept, sample, probs=q)
    wide = torch.full((12, 350), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:8, 3:336] = logits[:8].cuda()
    wide_q = torch.full((12, 340), float("nan"), device="cuda")
    wide_q[:8, 1:334] = q[:8].cuda()
    flat = torch.cat([_flat(parents), _i32([-5] * 4)])
    got = ops.verify_draft(wide[:, 3:336], drafts.cuda(), flat, _i32([0, 5, 8]), accept.cuda(), sample.cuda(),
                           draft_probs=wide_q[:, 1:334])
    assert [got[0].tolist(), got[1].tolist(), got[2][:8].tolist()] == [list(w) for w in want]
    ops.check_status(cuda_device)


def test_what_is_kept_has_the_targets_distribution(cuda_device) -> None:
    """200000 draws of one node's children and next token: the first token's frequencies are p. The sum of
    n p-hat's squared deviations over p is chi-square with 5 degrees of freedom: above 30 in 1.5e-5 of runs."""
    n, vocab = 200000, 6
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.tensor([0.3, -1.0, 1.2, 0.0, -0.5, 0.7])
    p = torch.softmax(logits.double(), 0)
    q = torch.softmax(torch.tensor([0.9, 0.1, 0.2, -0.4, 0.0, 0.5]).double(), 0).float()
    for probs in (True, False):
        drafts = torch.zeros(n, 3, dtype=torch.int64, device="cuda")
        if probs:
            drafts[:, 1:] = torch.multinomial(q.cuda(), 2 * n, replacement=True, generator=g).view(n, 2)
        else:
            drafts[:, 1:] = torch.tensor([2, 4], device="cuda")
        flat = drafts.view(-1)
        rows = 3 * n
        accepted, token, order = ops.verify_draft(
            logits.cuda().expand(rows, vocab).contiguous(), flat, _i32([-1, 0, 0]).repeat(n),
            torch.arange(0, rows + 1, 3, dtype=torch.int32, device="cuda"),
            torch.rand(rows, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g),
            draft_probs=q.cuda().expand(rows, vocab).contiguous() if probs else None)
        first = torch.where(accepted > 0, drafts[torch.arange(n, device="cuda"), order.view(n, 3)[:, 1].long()], token)
        count = torch.bincount(first, minlength=vocab).cpu().double()
        assert float(((count - n * p) ** 2 / (n * p)).sum()) < 30


def test_verify_refuses(cuda_device) -> None:
    case = _case([4], 50, probs=True, seed=1)
    good = dict(logits=case[1].cuda(), draft_tokens=case[2].cuda(), parents=_flat(case[0]), tree_start=_i32([0, 4]),
                accept_uniforms=case[3].cuda(), sample_uniforms=case[4].cuda(), draft_probs=case[5].cuda())
    bad = [dict(logits=good["logits"].half()), dict(logits=good["logits"][0]), dict(logits=good["logits"].t()),
           dict(draft_tokens=good["draft_tokens"].int()), dict(parents=good["parents"].long()),
           dict(parents=good["parents"][:3]), dict(tree_start=good["tree_start"].long()),
           dict(tree_start=good["tree_start"].cpu()), dict(accept_uniforms=None), dict(sample_uniforms=None),
           dict(accept_uniforms=good["accept_uniforms"].double()), dict(sample_uniforms=good["accept_uniforms"]),
           dict(draft_probs=good["draft_probs"].bfloat16()), dict(draft_probs=good["draft_probs"][:, :49]),
           dict(greedy=True), dict(temperature=0.0)]
    for change in bad:
        with pytest.raises(ValueError, match="verify_draft"):
            ops.verify_draft(**{**good, **change})
    none = ops.verify_draft(good["logits"], good["draft_tokens"], good["parents"], _i32([0]), good["accept_uniforms"],
                            good["sample_uniforms"][:0])
    assert none[0].numel() == 0 and none[1].numel() == 0


def test_verify_in_a_graph_and_on_a_side_stream(cuda_device) -> None:
    sizes = [7, 3, 12]
    cases = [_case(sizes, 3001, probs=True, seed=s) for s in (1, 2)]
    dev = [[_flat(c[0]), c[1].cuda(), c[2].cuda(), c[3].cuda(), c[4].cuda(), c[5].cuda()] for c in cases]
    static = [t.clone() for t in dev[0]]
    start = _i32(ref.starts(sizes))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = ops.verify_draft(static[1], static[2], static[0], start, static[3], static[4], draft_probs=static[5])
    for c, d in zip(cases, dev):
        for s, t in zip(static, d):
            s.copy_(t)
        for _ in range(2):
            graph.replay()
        want = ref.verify(c[1], c[2], c[0], c[3], c[4], probs=c[5])
        assert [t.tolist() for t in out] == [list(w) for w in want]
    assert _lib.launches > 0
