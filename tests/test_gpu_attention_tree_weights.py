"""The tree attention's weights go through the second product with fp32's accuracy, as the prefill attention's do."""

from __future__ import annotations

import pytest
import torch

from aios_b200.kernel import ops
from tests import draft_reference as ref
from tests.test_gpu_attention_tree import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("nodes", [3, 9, 50, 90])
@pytest.mark.parametrize("cached", [0, 20, 700])
def test_weights_are_not_rounded_to_bf16(cuda_device, d: int, nodes: int, cached: int) -> None:
    """Small scores and values of either sign, so that sums come out near 0 beside their terms. The result is rounded to
    bf16 (2^-8 of it), the weights' lower halves are (2^-8 of at most 2^-7 of the weight, and 2^-20 that is added to them);
    scores, exponentials and sums as in the general tolerance."""
    c = Case([nodes, 2], [cached, cached // 2], 4, 2, d, seed=d + nodes, spread=0.25)
    n = nodes + 2
    want, mag, top = ref.attention(c.q[:n], c.k, c.v, c.table, c.row_list, c.cached_list, c.sizes, c.mask[:n], 4, 2, d,
                                   c.scale)
    delta = 2 * (d + 4) * 2.0**-23 * top + ((cached + nodes) / 64 + 4) * 2.0**-21
    tol = (2.0**-15 + 2.0**-20 + 2 * delta) * mag * (1 + 2.0**-8) + 2.0**-8 * want.abs() + 1e-30
    for bound in (1, 1 << 20):
        got = c.run(max_cached=bound)
        err = (got[:n].double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
    ops.check_status(cuda_device)


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("nodes", [3, 50, 90])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_infinite_values_of_the_history(cuda_device, d: int, nodes: int, value: float) -> None:
    """Every node sees them: the column of each is what the value is, of either half of its weight, and others stay."""
    c = Case([nodes, 2], [700, 300], 4, 2, d, seed=d + nodes, spread=0.25)
    for bound in (1, 1 << 20):
        clean = c.run(max_cached=bound).view(nodes + 2, 4, d)
        kept = c.v.clone()
        for key, column in ((0, 5), (130, 6), (320, 7), (639, 8)):  # whole chunks of history
            c.v[int(c.table[c.row_list[0], key]), 1, column] = value
        got = c.run(max_cached=bound).view(nodes + 2, 4, d)
        c.v.copy_(kept)
        hit = got[:nodes, 2:, 5:9]
        assert bool((torch.isnan(hit) if value != value else hit == value).all())
        got[:nodes, 2:, 5:9] = clean[:nodes, 2:, 5:9]
        assert torch.equal(got, clean)
    ops.check_status(cuda_device)
