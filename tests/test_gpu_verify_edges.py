"""verify_draft at the edges of its inputs: weights next to nothing, rejections that leave little or nothing."""

from __future__ import annotations

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
