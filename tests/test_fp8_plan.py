"""Which kernel a linear's size runs on (``aiosb_linear_fp8_plan``, no GPU)."""

from __future__ import annotations

import pytest

from aios_b200 import _lib
from aios_b200.kernel import ops
from test_gpu_fp8 import EACH

PLANS = {(t, 128, s) for t in (16, 32, 64, 128) for s in (1, 2, 4, 8)} | {(256, 256, 1)}


def test_the_sizes_of_the_gpu_tests_reach_every_tile_and_split() -> None:
    assert {ops.linear_fp8_plan(*size, 148) for size in EACH} == PLANS


def test_plan_is_a_query() -> None:
    before = _lib.launches
    assert ops.linear_fp8_plan(1, 8192, 14336, 148)[0] == 16
    assert ops.linear_fp8_plan(8192, 8192, 8192, 148) == (256, 256, 1)
    assert _lib.launches == before
    for sms in (1, 2, 132, 1000):
        assert ops.linear_fp8_plan(77, 1000, 5008, sms) in PLANS
    for size, text in (((0, 8, 16), "no rows"), ((1, 4, 16), "multiple of 8"), ((1, 8, 24), "multiple of 16"),
                       ((1 << 31, 8, 16), "too large"), ((1, 8, 16, -1), "bad SM count")):
        with pytest.raises(ValueError, match=text):
            ops.linear_fp8_plan(*size)
    assert _lib.load().aiosb_linear_fp8_plan(1, 8, 16, 148, None) == _lib.ERR_INVALID_ARG
