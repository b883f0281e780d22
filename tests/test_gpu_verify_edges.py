"""verify_draft at the edges of its inputs: weights next to nothing, rejections that leave little or nothing."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from aios_b200.kernel import ops
from tests import draft_reference as ref

pytestmark = pytest.mark.gpu

INF = float("inf")


def _verify(logits, drafts, parents, accept, sample, probs=None, **kwargs):
    """One tree, node 0's row of logits (and probabilities) given; the other nodes' rows are the same."""
    n = len(parents)
    rows = torch.tensor(logits, dtype=torch.float32).expand(n, -1).contiguous()
    q = None if probs is None else torch.tensor(probs, dtype=torch.float32).expand(n, -1).contiguous()
    tokens, u, v = torch.tensor(drafts), torch.tensor(accept), torch.tensor([sample])
    args = [t.cuda() for t in (rows, tokens, torch.tensor(parents, dtype=torch.int32),
                               torch.tensor([0, n], dtype=torch.int32), u, v)]
    q_args = None if q is None else q.cuda()
    junk = [torch.full((1,), 1 << 40, dtype=torch.int64, device="cuda") for _ in range(4)]
    del junk  # an output that is left unwritten holds this
    got = ops.verify_draft(*args, draft_probs=q_args, **kwargs)
    want = ref.verify(rows, tokens, [parents], u, v, probs=q, **kwargs)
    return [t.tolist() for t in got], [list(w) for w in want]


def _spread(values: list[float], vocab: int) -> list[float]:
    """The values at equal distances among masked tokens, so that they fall to different CTAs of a request."""
    row = [-INF] * vocab
    for i, x in enumerate(values):
        row[i * (vocab // len(values)) + 3] = x
    return row


@pytest.mark.parametrize("vocab", [8, 9000, 70000])
@pytest.mark.parametrize("below", [500.0, 556.0, 580.0, 599.0])
def test_tokens_up_to_600_temperatures_below_the_largest(cuda_device, vocab: int, below: float) -> None:
    """A rejection of the only likely token (a uniform above 1 forces it) leaves tokens of tiny weights: they are
    drawn from, as those that lie no more than 600 temperatures below the largest."""
    for temperature in (1.0, 0.25):
        logits = _spread([0.0, -below * temperature, -(below + 0.5) * temperature], vocab)
        at = [i for i, x in enumerate(logits) if x > -INF]
        for sample in (0.3, 0.7):
            got, want = _verify(logits, [0, at[0]], [-1, 0], [0.0, 1.5], sample, temperature=temperature)
            assert want[1][0] == at[1 if sample < 0.6 else 2]  # 1 / (1 + e^-0.5) = 0.62
            assert got == want
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [1, 8, 70000])
@pytest.mark.parametrize("u", [1.0, 1.5])
def test_a_rejection_that_would_leave_nothing(cuda_device, vocab: int, u: float) -> None:
    """Without probabilities: a forced token, rejected by a uniform of 1 (splitmix uniforms round up to it), stays the
    only one, for later children and as the next token."""
    logits = [-INF] * vocab
    x = vocab - 1
    logits[x] = 3.0
    for parents, drafts, accept, accepted, token in [
        ([-1, 0], [0, x], [0.0, u], 0, x),
        ([-1, 0, 0, 0], [0, x, 0, x], [0.0, u, u, 0.5], 1 if vocab > 1 else None, x),
        ([-1, 0, 0, 0], [0, x, 0, x], [0.0, u, u, u], 0, x),
        ([-1] + [0] * 70, [0] + [x] * 70, [0.0] + [u] * 66 + [0.9] * 4, 1, x),
        ([-1] + [0] * 70, [0] * 36 + [x] * 35, [0.0] + [u] * 70, 0, x),
    ]:
        got, want = _verify(logits, drafts, parents, accept, 0.4)
        assert got == want and got[1] == [token] and accepted in (None, got[0][0])
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [24, 70000])
@pytest.mark.parametrize("step", [15.7, 16.2])
def test_what_near_certain_rejections_leave(cuda_device, vocab: int, step: float) -> None:
    """Children that have all but e^-16 of what is left, one after another, each rejected by a uniform next to 1: the
    last one is tried against its share of a sum that is 2^-69 of the first."""
    logits = _spread([0.0, -step, -2 * step, -3 * step, -3 * step - 0.7, -3 * step - 0.9], vocab)
    at = [i for i, x in enumerate(logits) if x > -INF]
    share = 1 / (1 + 2.718281828459045**-0.7 + 2.718281828459045**-0.9)
    below = 1 - 2.0**-24
    for u in (share - 0.1, share - 1e-4, share + 1e-4, share + 0.1, below):
        for sample in (0.3, 0.5, 0.6):
            got, want = _verify(logits, [0] + at[:4], [-1] + [0] * 4, [0.0] + [below] * 3 + [u], sample)
            assert want[0] == [1 if u < share else 0]
            assert got == want
    ops.check_status(cuda_device)


def test_many_proposals_of_few_tokens(cuda_device) -> None:
    """Tokens repeated among up to 200 children, within and across groups of 32: each counts once."""
    g = torch.Generator().manual_seed(9)
    for n in (2, 31, 33, 64, 65, 200):
        for vocab in (5, 40, 300):
            logits = (2 * torch.randn(vocab, generator=g)).tolist()
            for top in (1.0, 0.99999):
                drafts = [0] + torch.randint(0, vocab, (n,), generator=g).tolist()
                accept = [0.0] + (1 - torch.rand(n, generator=g) ** 4 * top).tolist()
                got, want = _verify(logits, drafts, [-1] + [0] * n, accept, 0.5)
                assert got == want


@pytest.mark.parametrize("vocab", [8, 9000, 70000])
@pytest.mark.parametrize("below", [60.0, 95.0, 400.0, 599.0])
def test_what_the_drafting_model_never_proposes_loses_nothing(cuda_device, vocab: int, below: float) -> None:
    """Probabilities of 0 take nothing, not even from the smallest of weights."""
    logits = _spread([0.0, -below, -below - 0.5], vocab)
    at = [i for i, x in enumerate(logits) if x > -INF]
    for zero in (0.0, -0.0):
        q = [zero] * vocab
        q[at[0]] = 1.0
        for sample in (0.3, 0.7):
            got, want = _verify(logits, [0, at[0]], [-1, 0], [0.0, 1.5], sample, q)
            assert want[1][0] == at[1 if sample < 0.6 else 2]  # 1 / (1 + e^-0.5) = 0.62
            assert got == want
    ops.check_status(cuda_device)


@pytest.mark.parametrize("zero", [0.0, -0.0, 1e-39])
def test_a_masked_token_gains_nothing(cuda_device, zero: float) -> None:
    """q = p but for the sign of a masked token's 0 (or a probability that is none of the normal numbers): nothing is
    left, so the distribution stays."""
    for sample, token in ((0.2, 0), (0.6, 1), (0.99, 1)):
        got, want = _verify([0.0, 0.0, -INF], [0, 0], [-1, 0], [0.0, 1.5], sample, [0.5, 0.5, zero])
        assert got == want and got[1] == [token]
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [6, 70000])
@pytest.mark.parametrize("value", [float("nan"), -float("nan"), INF, -INF])
def test_probabilities_that_are_none(cuda_device, vocab: int, value: float) -> None:
    """Seen where they are read: at a child's own token, and in the row that a rejection takes off. The path ends there
    without a next token, as it does at a row of logits that is no distribution."""
    x = vocab - 2
    logits = [0.0] * vocab
    q = [1.0 / vocab] * vocab
    q[x] = value
    for drafts, accept, stays in (([0, x], [0.0, 0.1], 0), ([0, 1], [0.0, 5.0 * vocab], 0),
                                  ([0, 1, x], [0.0, 5.0 * vocab, 0.1], 0)):
        got, _ = _verify(logits, drafts, [-1] + [0] * (len(drafts) - 1), accept, 0.5, q)
        assert got[0] == [stays] and got[1] == [-1] and got[2] == list(range(len(drafts)))
        with pytest.raises(RuntimeError, match="no token"):
            ops.check_status(cuda_device)
    # not read: the first child stays, and its own row has no children
    got, _ = _verify(logits, [0, 1], [-1, 0], [0.0, 0.5], 0.5, q)
    assert got[0] == [1] and 0 <= got[1][0] < vocab
    ops.check_status(cuda_device)


def test_probabilities_are_taken_as_they_are(cuda_device) -> None:
    """Above 1 or below 0, they go into the formula all the same."""
    for x, value in ((2, -0.25), (2, 7.0), (3, -1e-30)):
        q = [0.2, 0.3, 0.1, 0.4]
        q[x] = value
        for sample in (0.1, 0.4, 0.7, 0.95):
            for accept in (0.1, 3.0):
                got, want = _verify([0.5, 0.1, 0.2, -0.3], [0, 1, 2], [-1, 0, 0], [0.0, 3.0, accept], sample, q)
                assert got == want
    ops.check_status(cuda_device)


def _temperature_for(u: float, lower: float, nudge: float) -> float:
    """Where a token 0 has the share u * (1 + nudge) beside one of logit -lower."""
    share = u * (1 + nudge)
    return lower / math.log(share / (1 - share))


def test_borders_between_ctas(cuda_device) -> None:
    """The likeliest two tokens in different CTAs of a request, |logit| / T about 10^7: fp64's rounding of logit / T must
    not come between them. The draws lie 5e-11 to 1e-10 of the sum from the border; the temperatures are those where
    twice the roundings (of 16 logit / (T ln 2), exact by fractions) would carry the border across."""
    vocab, found = 70000, 0
    for m1 in (20.0, -20.0, 300.0):
        m2 = float(torch.nextafter(torch.tensor(m1), torch.tensor(-INF)))
        row = [-INF] * vocab
        row[3], row[60003] = m1, m2
        for i in range(400):
            nudge = (5e-11 + 5e-11 * i / 400) * (1 if i % 2 else -1)
            t = _temperature_for(0.75, m1 - m2, nudge)
            scale = (1 / t) * (1.4426950408889634 * 16)
            e1, e2 = (float(Fraction(m) * Fraction(scale) - Fraction(m * scale)) for m in (m1, m2))
            crossed = 0.25 * (e1 - e2) * math.log(2) / 16 * (1 if nudge < 0 else -1)
            if crossed < 1.5 * abs(nudge):
                continue
            found += 1
            got, want = _verify(row, [0], [-1], [0.0], 0.75, temperature=t)
            assert want[1] == [3 if nudge > 0 else 60003]
            assert got == want
            if found % 8 == 0:
                break
    assert found >= 16


@pytest.mark.parametrize("probs", [False, True])
def test_borders_within_fp64(cuda_device, probs: bool) -> None:
    """Draws 2e-14 of the sum from a border, for weights anywhere between the table's entries: those in the middle are
    where an exponential of less than fp64's digits is off by most."""
    for eighth in range(100, 125):
        z = eighth / 4 * math.log(2) / 16 + 1e-4
        u = float(torch.tensor(1 / (1 + math.exp(-z))))
        for nudge in (-2e-14, 2e-14):
            t = _temperature_for(u, 1.0, nudge)
            got, want = _verify([0.0, -1.0], [0], [-1], [0.0], u, [0.5, 0.5] if probs else None, temperature=t)
            assert want[1] == [0 if nudge > 0 else 1]
            assert got == want, (eighth, nudge)


@pytest.mark.parametrize("mode", ["greedy", "plain", "probs"])
@pytest.mark.parametrize("node,parent", [(2, 2), (1, 3), (3, -2), (2, 1 << 20), (0, 0), (1, -(1 << 31))])
def test_parents_that_are_no_earlier_node_are_reported(cuda_device, mode: str, node: int, parent: int) -> None:
    """As by draft_tree: the node counts as a root, so nothing leads to it."""
    parents, drafts = [-1, 0, 0, 1], [0, 3, 4, 2]
    logits = [0.0, 0.1, 0.3, 0.9, 0.2]
    q = [0.2] * 5 if mode == "probs" else None
    kw = {"greedy": True} if mode == "greedy" else {}
    as_root = [-1 if i == node else p for i, p in enumerate(parents)]
    want, _ = _verify(logits, drafts, as_root, [0.0, 0.3, 0.3, 0.3], 0.5, q, **kw)
    ops.check_status(cuda_device)
    got, _ = _verify(logits, drafts, [parent if i == node else p for i, p in enumerate(parents)],
                     [0.0, 0.3, 0.3, 0.3], 0.5, q, **kw)
    assert got == want
    with pytest.raises(RuntimeError, match="tree"):
        ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [8, 70000])
def test_the_smallest_probabilities(cuda_device, vocab: int) -> None:
    """Subnormal ones count as they are: e^-150 less 2^-147 is nothing, e^-95 less 2^-140 is not."""
    for lower, q1, left in ((150.0, 2.0**-147, False), (95.0, 2.0**-140, True), (101.0, 2.0**-149, True),
                            (101.0, 2.0**-145, False), (101.0, 0.0, True)):
        logits = _spread([0.0, -lower], vocab)
        at = [i for i, x in enumerate(logits) if x > -INF]
        q = [0.0] * vocab
        q[at[0]], q[at[1]] = 1.0, q1
        got, want = _verify(logits, [0, at[0]], [-1, 0], [0.0, 1.5], 0.5, q)
        assert got == want and got[1] == [at[1] if left else at[0]]
    ops.check_status(cuda_device)


@pytest.mark.parametrize("vocab", [16, 70000])
def test_what_a_certain_drafting_model_leaves(cuda_device, vocab: int) -> None:
    """A drafting model that is certain of the token that the target is all but certain of: a rejection (of a masked
    token) takes all of it, whatever the logit's size, and the rest is left."""
    for largest in (0.1, 20.3, -47.7, 301.0):
        for temperature in (1.0, 0.05, 0.3):
            logits = _spread([largest, largest - 100 * temperature, largest - 100.5 * temperature, -INF], vocab)
            at = [i * (vocab // 4) + 3 for i in range(4)]
            q = [0.0] * vocab
            q[at[0]] = 1.0
            for sample in (0.3, 0.7):
                got, want = _verify(logits, [0, at[3]], [-1, 0], [0.0, 0.5], sample, q, temperature=temperature)
                assert got == want and got[1] == [at[1 if sample < 0.6 else 2]]  # 1 / (1 + e^-0.5) = 0.62
    ops.check_status(cuda_device)
