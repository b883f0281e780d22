"""The 8-bit operators on operands at the ends of their ranges, against 64 bits.

Bounds as in test_gpu_fp8.py; an output below 2^-126 is bf16's subnormal, half a step 2^-134.
"""

from __future__ import annotations

import pytest
import torch

from aios_b200 import _lib
from aios_b200.kernel import ops
from test_fp8_plan import PLANS
from test_gpu_fp8 import BLOCK, EACH, _linear_check, _linear_inputs, _values

pytestmark = pytest.mark.gpu


def _operands(rows: int, n: int, k: int):
    """Ordinary e4m3 rows and weight with scales as a model has them."""
    g = torch.Generator("cuda").manual_seed(rows + n + k)
    blocks = -(-k // BLOCK)

    def values(m):
        v = torch.empty(m, k, device="cuda").normal_(std=60.0, generator=g).clamp(-448, 448)
        return v.to(torch.float8_e4m3fn)

    def scales(m):
        return torch.empty(m, blocks, device="cuda").uniform_(0.002, 0.01, generator=g)

    return values(rows), scales(rows), values(n), scales(-(-n // BLOCK))


def _check(y, q, s, wq, ws) -> None:
    x, w = _values(q, s), _values(wq, ws, BLOCK)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    terms = BLOCK + -(-q.shape[1] // BLOCK)
    bad = ~((y.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-134 + 2.0**-23 * terms * size)
    assert not bool(bad.any()), f"{int(bad.sum())} values off, first at {bad.nonzero()[0].tolist()}"


def test_this_device_runs_every_tile_and_split(cuda_device) -> None:
    assert {ops.linear_fp8_plan(*size) for size in EACH} == PLANS


# more tiles than pairs of SMs, k in an odd number of groups of eight blocks: the order of the scale
# buffers goes on from tile to tile
@pytest.mark.parametrize("rows,n,k", [(3000, 2600, 2352), (2500, 3000, 2640), (4100, 4104, 400)])
def test_pairs_that_walk_several_tiles(cuda_device, rows: int, n: int, k: int) -> None:
    assert ops.linear_fp8_plan(rows, n, k) == (256, 256, 1)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-rows // 256) * -(-n // 256) > sms // 2
    q, s, wq, ws = _linear_inputs(rows, n, k)
    y = ops.linear_fp8(q, s, wq, ws)
    _linear_check(y, q, s, wq, ws)
    r = torch.randn(rows, n, device=cuda_device).to(torch.bfloat16)
    z = ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_ADD, residual=r)
    _linear_check(z, q, s, wq, ws, r)
    ops.check_status(cuda_device)


@pytest.mark.parametrize("rows,n,k", [*EACH, (3000, 2600, 2352)])
def test_scales_whose_product_fp32_does_not_hold(cuda_device, rows: int, n: int, k: int) -> None:
    """2^70 x 2^60 overflows and 1.3 x 2^-78 x 1.2 x 2^-70 is left with two bits, 2^-82 x 2^-70 with none;
    the sums are ordinary numbers."""
    q, s, wq, ws = _operands(rows, n, k)
    last = -(-k // BLOCK) - 1
    q8, w8 = q.view(torch.uint8), wq.view(torch.uint8)
    edge = ws.shape[0] // 2  # the features whose weight scales are extreme in the first and the last block
    large = torch.arange(rows, device="cuda") % 5 == 1
    small = torch.arange(rows, device="cuda") % 5 == 2
    empty = torch.arange(rows, device="cuda") % 5 == 3
    plain = ~(large | small | empty)
    ws[edge, 0], ws[edge, last] = 2.0**60, 1.2 * 2.0**-70
    w8[:, 0] = torch.where(w8[:, 0] > 0x7F, 0x89, 0x09)  # +-2^-6 x 1.125
    before = ops.linear_fp8(q, s, wq, ws)
    # overflow: one value of 2^-9 in the first block, times 2^70; nothing at all in some of the rows
    q8[large, :BLOCK] = 0
    q8[large & (torch.arange(rows, device="cuda") % 2 == 0), 0] = 0x01
    s[large, 0] = 2.0**70
    # underflow: rows that are 448 in the last block and empty elsewhere
    q8[small, : last * BLOCK] = 0
    q8[small, last * BLOCK :] = 0x7E
    s[small, last] = torch.where(torch.arange(int(small.sum()), device="cuda") % 2 == 0, 1.3 * 2.0**-78, 2.0**-82)
    # empty rows, whose scales some quantisers leave at 0
    q8[empty] = 0
    s[empty] = 0
    y = ops.linear_fp8(q, s, wq, ws)
    _check(y, q, s, wq, ws)
    assert torch.equal(y[plain], before[plain])  # a row's bits do not depend on its neighbours' scales
    assert torch.equal(y, ops.linear_fp8(q, s, wq, ws, stable_weight=True))
    ops.check_status(cuda_device)


@pytest.mark.parametrize("rows", [8, 24, 60, 200, 1500])
def test_every_pair_of_extreme_scales(cuda_device, rows: int) -> None:
    """One value of 1 to a row, in the second of three blocks: an output is the product of its two scales."""
    ends = [0.0, 2.0**-149, 2.0**-120, 2.0**-60, 1.0, -(2.0**60), 2.0**110, 3e38, float("inf"), float("nan")]
    n, k = BLOCK * len(ends), 3 * BLOCK
    q = torch.zeros(rows, k, device="cuda")
    q[:, BLOCK + 7] = 1
    wq = torch.zeros(n, k, device="cuda")
    wq[:, BLOCK + 7] = 1
    s, ws = torch.ones(rows, 3, device="cuda"), torch.ones(len(ends), 3, device="cuda")
    s[:, 1] = torch.tensor(ends, device="cuda").repeat(-(-rows // len(ends)))[:rows]
    ws[:, 1] = torch.tensor(ends, device="cuda")
    y = ops.linear_fp8(q.to(torch.float8_e4m3fn), s, wq.to(torch.float8_e4m3fn), ws).double()
    want = s[:, 1, None].double() * ws[:, 1].double().repeat_interleave(BLOCK)
    over = want.abs() >= 2.0**128
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y[over], torch.where(want[over] > 0, float("inf"), -float("inf")))
    rest = ~over & ~want.isnan()
    bad = (y - want).abs()[rest] > 2.0**-8 * want[rest].abs() + 2.0**-134 + 2.0**-149
    assert not bool(bad.any())


def _every_operator(rows: int = 13, width: int = 784):
    x = torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(torch.bfloat16)
    r, g = x.flip(0).contiguous(), x[0].contiguous()
    wq, ws = ops.quantize_weight_fp8(x[:8].contiguous())
    q, s = ops.quantize_fp8(x)
    out = [q, s, wq, ws, *ops.rmsnorm_fp8(x, g, 1e-6), *ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6), r]
    out += [*ops.silu_and_mul_fp8(x[:, : width - 16]), ops.linear_fp8(q, s, wq, ws)]
    return [t.view(torch.uint8) if t.dtype is ops.FP8_DTYPE else t for t in out]


def test_outputs_do_not_depend_on_how_they_are_allocated(cuda_device, monkeypatch) -> None:
    """The allocator's short entry, its fallback, and the fill of fresh memory that deterministic mode asks for."""
    want = _every_operator()
    monkeypatch.setattr(ops, "_new_cuda", None)
    got = _every_operator()
    torch.use_deterministic_algorithms(True)
    try:
        filled = _every_operator()
    finally:
        torch.use_deterministic_algorithms(False)
    for a, b, c in zip(want, got, filled):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
        assert torch.equal(a, b) and torch.equal(a, c)


def test_single_rows_of_wide_buffers(cuda_device) -> None:
    """One row has no stride; its buffers' rows may be any distance apart."""
    q, s, wq, ws = _linear_inputs(1, 264, 784)
    wide = torch.zeros(3, 1008, dtype=torch.uint8, device=cuda_device)
    wide[1:2, 16:800] = q.view(torch.uint8)
    x = wide.view(ops.FP8_DTYPE)[1:2, 16:800]
    want = ops.linear_fp8(q, s, wq, ws)
    buf = torch.full((3, 500), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    out = buf[1:2, 4:268]  # row 1 begins 1000 bytes in: 16-byte aligned from its fifth value on
    r = torch.randn(1, 264, device=cuda_device).to(torch.bfloat16)
    ops.linear_fp8(q, s, wq, ws, out=out, epilogue=_lib.EPI_ADD, residual=r)
    _linear_check(out, q, s, wq, ws, r)
    assert int(buf.isnan().sum()) == buf.numel() - 264
    assert torch.equal(ops.linear_fp8(x, s, wq, ws), want)


@pytest.mark.parametrize("rows,n,k", [(100001, 8, 16), (70000, 72, 144), (1, 100008, 16)])
def test_thin_linears(cuda_device, rows: int, n: int, k: int) -> None:
    q, s, wq, ws = _linear_inputs(rows, n, k)
    y = ops.linear_fp8(q, s, wq, ws)
    _linear_check(y, q, s, wq, ws)
    assert torch.equal(y, ops.linear_fp8(q, s, wq, ws, stable_weight=True))
    ops.check_status(cuda_device)


def test_operands_that_are_the_same_tensor(cuda_device) -> None:
    """x + x in place, the sum written over x, and a weight that is its own input."""
    x = torch.randn(40, 784, device=cuda_device).to(torch.bfloat16)
    g = torch.ones(784, dtype=torch.bfloat16, device=cuda_device)
    want = ops.rmsnorm_fp8((2 * x.float()).to(torch.bfloat16), g, 4e-6)
    a = x.clone()
    q, s = ops.fused_add_rmsnorm_fp8(a, a, g, 4e-6)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])
    assert torch.equal(a, (2 * x.float()).to(torch.bfloat16))
    b, r = x.clone(), x.flip(0).contiguous()
    q, s = ops.fused_add_rmsnorm_fp8(b, r, g, 1e-6, residual_out=b)
    q2, s2 = ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6, residual_out=torch.empty_like(x))
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    assert torch.equal(b, (x.float() + r.float()).to(torch.bfloat16)) and torch.equal(r, x.flip(0))
    wq, ws = ops.quantize_weight_fp8(x)
    xq, xs = ops.quantize_fp8(x)
    _linear_check(ops.linear_fp8(wq, xs, wq, ws), wq, xs, wq, ws)
