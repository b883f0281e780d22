"""The 8-bit linear operators on the GPU against their definitions in 64 bits.

A value v of a block with scale s becomes q with |q * s - v| <= 2^-4 |v| (half a step of
e4m3's three mantissa bits, relative) or 2^-10 s (half its subnormal step), whichever is
larger, once v itself is off by a relative `slack` from fp32 arithmetic:

* quantisers: v is the bf16 input; one division and one product, 2 x 2^-24: slack 2^-22.
  Every step is an IEEE operation, so the bytes equal those of the same formula in torch.
* norm: at most 32 serial and 10 tree additions of squares (each 2^-24, halved by the
  root), a division, a root, two products: under 64 x 2^-24: slack 2^-18.
* SwiGLU: the hardware exponential is off by 2 + 1.173 |g| units of 2^-23, at most 105 of
  them for |g| <= 87, the division and products by a few more: slack 2^-16.

Linear: bf16 rounding 2^-8 |y| (half a step) and fp32 sums over k, each of at most
128 + ceil(k / 128) additions of terms bounded by sum |x w|: 2^-23 (128 + ceil(k / 128)) sum |x w|.
"""

from __future__ import annotations

import pytest
import torch

from aios_b200 import _lib
from aios_b200.kernel import ops

pytestmark = pytest.mark.gpu

BLOCK = 128


def _spread(scale: torch.Tensor, tall: int, rows: int, cols: int) -> torch.Tensor:
    s = scale.double().repeat_interleave(BLOCK, dim=1)[:, :cols]
    return s if tall == 1 else s.repeat_interleave(tall, dim=0)[:rows]


def _values(q: torch.Tensor, scale: torch.Tensor, tall: int = 1) -> torch.Tensor:
    return q.double() * _spread(scale, tall, *q.shape)


def _amax(v: torch.Tensor, tall: int) -> torch.Tensor:
    rows, cols = v.shape
    rb, cb = -(-rows // tall), -(-cols // BLOCK)
    p = torch.zeros(rb * tall, cb * BLOCK, dtype=v.dtype, device=v.device)
    p[:rows, :cols] = v
    return p.view(rb, tall, cb, BLOCK).abs().amax(dim=(1, 3))


def _check_quantised(q, scale, v, slack: float, tall: int = 1) -> None:
    """q * scale against the 64-bit values v."""
    want = torch.clamp(_amax(v, tall), min=2.0**-100) / 448
    assert scale.shape == want.shape and scale.dtype == torch.float32 and q.dtype == torch.float8_e4m3fn
    assert bool(((scale.double() - want).abs() <= want * (slack + 2.0**-24)).all())
    err = (_values(q, scale, tall) - v).abs()
    bound = torch.maximum(2.0**-4 * v.abs(), 2.0**-10 * _spread(scale, tall, *v.shape)) * (1 + slack) + slack * v.abs()
    bad = err > bound
    assert not bool(bad.any()), f"{int(bad.sum())} values off, first at {bad.nonzero()[0].tolist()}"


def _rows(rows: int, cols: int, seed: int, width: int | None = None, device="cuda") -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width or cols, generator=g) * torch.exp(torch.randn(1, width or cols, generator=g))
    x[5::7] = 0  # empty rows
    return x.to(torch.bfloat16).to(device)[:, :cols]


SHAPES = [(1, 16), (1, 768), (3, 128), (8, 144), (13, 768), (33, 2000), (257, 1008), (64, 2048), (5, 4096), (9, 5120),
          (17, 8192), (4, 12304), (3, 16384), (2, 20496), (2, 32768)]


@pytest.mark.parametrize("pad", [0, 24])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_rows_bits(cuda_device, rows: int, cols: int, pad: int) -> None:
    x = _rows(rows, cols, rows + cols, cols + pad)
    q, s = ops.quantize_fp8(x)
    _check_quantised(q, s, x.double(), 2.0**-22)
    amax = torch.clamp(_amax(x.float(), 1), min=2.0**-100)
    top = torch.full_like(amax, 448)  # a tensor: torch divides by a number through its reciprocal
    inv = (top / amax).repeat_interleave(BLOCK, dim=1)[:, :cols]
    assert torch.equal(s, amax / top)
    assert torch.equal((x.float() * inv).to(torch.float8_e4m3fn).view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("n,k", [(1, 16), (8, 128), (127, 144), (128, 768), (1280, 768), (1000, 2000), (130, 8208)])
def test_quantize_weight_bits(cuda_device, n: int, k: int) -> None:
    w = _rows(n, k, n + k, k + 8)
    q, s = ops.quantize_weight_fp8(w)
    _check_quantised(q, s, w.double(), 2.0**-22, tall=BLOCK)
    amax = torch.clamp(_amax(w.float(), BLOCK), min=2.0**-100)
    top = torch.full_like(amax, 448)
    inv = (top / amax).repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    assert torch.equal(s, amax / top)
    assert torch.equal((w.float() * inv).to(torch.float8_e4m3fn).view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rmsnorm_fp8(cuda_device, rows: int, cols: int, residual: bool) -> None:
    x = _rows(rows, cols, 3 * rows + cols, cols + 16)
    g = (1 + 0.1 * torch.randn(cols, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).to(cuda_device)
    s = x.double()
    if residual:
        r = _rows(rows, cols, 7 * rows + cols).contiguous()
        s = s + r.double()
        before = r.clone()
        r_out = torch.empty_like(r)
        q, scale = ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6, residual_out=r_out)
        assert torch.equal(r, before)
        assert torch.equal(r_out, (x.float() + r.float()).to(torch.bfloat16))  # the sum of two bf16 rounds once
        q2, scale2 = ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6)  # in place
        assert torch.equal(r, r_out) and torch.equal(scale, scale2)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    else:
        q, scale = ops.rmsnorm_fp8(x, g, 1e-6)
    v = s / torch.sqrt(s.square().mean(dim=1, keepdim=True) + 1e-6) * g.double()
    _check_quantised(q, scale, v, 2.0**-18)


# the last two: two and four groups of 128 columns to 16 lanes
@pytest.mark.parametrize("rows,f", [(1, 16), (8, 2048), (13, 144), (257, 1008), (3, 10240), (1000, 128), (3001, 1040),
                                    (5001, 2576)])
def test_silu_and_mul_fp8(cuda_device, rows: int, f: int) -> None:
    x = _rows(rows, 2 * f, rows + f, 2 * f + 8)
    q, s = ops.silu_and_mul_fp8(x)
    g, u = x[:, :f].double(), x[:, f:].double()
    v = g * torch.sigmoid(g) * u
    v[g < -87] = 0  # documented: a gate below -87 gives 0
    _check_quantised(q, s, v, 2.0**-16)


def test_silu_and_mul_fp8_of_extreme_gates(cuda_device) -> None:
    """One gate to a block of 128, times a factor that brings small results back into range."""
    gates = [0.0, -0.0, 1e-30, 20.0, 88.5, 3e38, -1.0, -20.0, -60.0, -86.5, -88.0, -100.0, -3e38]
    x = torch.zeros(1, 2 * BLOCK * len(gates), dtype=torch.bfloat16, device=cuda_device)
    f = BLOCK * len(gates)
    for i, g in enumerate(gates):
        x[0, i * BLOCK + 5] = g
        x[0, f + i * BLOCK + 5] = 0.5 if g > 1 else 1e30 if g > -30 else 1e38
    q, s = ops.silu_and_mul_fp8(x)
    g, u = x[:, :f].double(), x[:, f:].double()
    v = g / (1 + torch.exp(-g)) * u
    v[g < -87] = 0  # documented: a gate below -87 gives 0
    _check_quantised(q, s, v, 2.0**-16)
    x[0, 5], x[0, BLOCK + 5], x[0, 2 * BLOCK + 5] = float("inf"), float("-inf"), float("nan")
    q, s = ops.silu_and_mul_fp8(x)
    assert float(s[0, 0]) == float("inf") and bool(s[0, 1:3].isnan().all()) and bool(s[0, 3:].isfinite().all())


def _linear_check(y, q, s, wq, ws, residual=None) -> None:
    x, w = _values(q, s), _values(wq, ws, BLOCK)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    if residual is not None:
        want = want + residual.double()
    terms = BLOCK + -(-q.shape[1] // BLOCK)
    bad = (y.double() - want).abs() > 2.0**-8 * want.abs() + 2.0**-23 * terms * size
    assert not bool(bad.any()), f"{int(bad.sum())} values off, first at {bad.nonzero()[0].tolist()}"


def _linear_inputs(rows: int, n: int, k: int):
    q, s = ops.quantize_fp8(_rows(rows, k, rows + k))
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(n + k)) * 0.02).to(torch.bfloat16).cuda()
    return q, s, *ops.quantize_weight_fp8(w)


def _wide(n: int, k: int):
    """A quantised weight made in place on the device, for sizes that the host would be slow to make."""
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    w.normal_(std=0.02, generator=torch.Generator("cuda").manual_seed(n))
    return ops.quantize_weight_fp8(w)


# Sizes that the estimate gives to each kernel: 16, 32 and 64 tokens to a tile, 128 x 128 tiles,
# the pair of SMs; k whole and split in 2, 4 and 8; tiles cut by rows, n and k.
LINEARS = [(r, n, k) for r in (1, 8, 33, 128, 129, 300) for n, k in ((8, 16), (136, 144), (1280, 768), (776, 2064))]
LINEARS += [(1, 4104, 1024), (77, 1000, 5008), (64, 128, 8192), (500, 4096, 768), (1024, 2440, 144), (1100, 2432, 768),
            (2048, 2568, 144), (2040, 2560, 1040), (4096, 4096, 272), (513, 16384, 768), (16, 104, 128),
            (17, 10000, 1040), (40, 776, 8192)]
LINEARS += [(1, 8192, 1680), (5, 4096, 2064), (40, 4096, 1680), (40, 2056, 2064), (50, 16384, 400), (64, 8192, 4096),
            (40, 4096, 2064), (50, 2056, 8192), (77, 8192, 400), (77, 2056, 4096), (3, 776, 1040), (40, 16384, 1040),
            (100, 8192, 4096), (50, 4096, 8192), (77, 2056, 8192), (128, 16384, 400), (200, 8192, 400)]


@pytest.mark.parametrize("rows,n,k", LINEARS)
def test_linear_fp8(cuda_device, rows: int, n: int, k: int) -> None:
    q, s, wq, ws = _linear_inputs(rows, n, k)
    y = ops.linear_fp8(q, s, wq, ws)
    torch.cuda.synchronize()
    ops.check_status(cuda_device)
    _linear_check(y, q, s, wq, ws)
    # the order of the sums depends on the sizes alone, and an early fetched weight is the same weight
    assert torch.equal(y, ops.linear_fp8(q, s, wq, ws))
    assert torch.equal(y, ops.linear_fp8(q, s, wq, ws, stable_weight=True))


@pytest.mark.parametrize("rows,n,k", [(1, 768, 2048), (8, 768, 768), (130, 1000, 272), (2048, 2560, 528),
                                         (2040, 2568, 272), (1100, 2440, 528), (4100, 4104, 144), (77, 8200, 144)])
def test_linear_fp8_add_and_strides(cuda_device, rows: int, n: int, k: int) -> None:
    q, s, wq, ws = _linear_inputs(rows, n, k)
    wide = torch.zeros(rows, k + 48, dtype=torch.uint8, device=cuda_device)
    wide[:, :k] = q.view(torch.uint8)
    wide[:, k:] = 0x7F  # NaN beside every row
    xv = wide.view(torch.float8_e4m3fn)[:, :k]
    buf = torch.randn(rows + 1, n + 16, device=cuda_device).to(torch.bfloat16)
    before = buf.clone()
    out = buf[:rows, :n]
    y = ops.linear_fp8(xv, s, wq, ws, epilogue=_lib.EPI_ADD, residual=out, out=out)
    assert y.data_ptr() == out.data_ptr()
    _linear_check(y, q, s, wq, ws, before[:rows, :n])
    assert torch.equal(buf[:, n:], before[:, n:]) and torch.equal(buf[rows:], before[rows:])  # nothing beside it


# One size or more for each tile and each split of k, with and without a residual (instances
# of their own): 16-, 32- and 64-token tiles, 128 x 128 (also several to a CTA), the pair.
EACH = [(3, 1064, 560), (1, 4280, 1696), (8, 2288, 4432), (13, 552, 2112), (16, 264, 4512)]
EACH += [(18, 72, 144), (355, 272, 1760), (45, 1040, 2720), (18, 488, 2528), (21, 64, 1568)]
EACH += [(957, 520, 160), (482, 608, 3760), (80, 1584, 4704), (35, 1056, 5936)]
EACH += [(1370, 824, 144), (359, 3096, 1472), (947, 576, 2160), (34, 2112, 1872), (355, 264, 10032), (43, 912, 7888)]
EACH += [(795, 1424, 416), (216, 6664, 1808), (693, 792, 3472), (633, 424, 5216), (66, 1440, 7312)]
EACH += [(711, 3152, 144), (459, 616, 2448), (150, 2456, 4560), (2242, 1056, 528), (284, 8432, 2736)]
EACH += [(2500, 1400, 272), (300, 16392, 144)]


@pytest.mark.parametrize("rows,n,k", EACH)
def test_each_tile_and_split_with_and_without_residual(cuda_device, rows: int, n: int, k: int) -> None:
    q, s, wq, ws = _linear_inputs(rows, n, k)
    y = ops.linear_fp8(q, s, wq, ws)
    _linear_check(y, q, s, wq, ws)
    r = torch.randn(rows, n + 8, device=cuda_device).to(torch.bfloat16)[:, :n]
    z = ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_ADD, residual=r)
    _linear_check(z, q, s, wq, ws, r)
    buf = torch.full((rows + 1, n + 16), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    buf[:rows, :n] = r
    ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_ADD, residual=buf[:rows, :n], out=buf[:rows, :n])
    assert torch.equal(buf[:rows, :n], z)
    assert bool(buf[:, n:].isnan().all()) and bool(buf[rows:].isnan().all())  # nothing beside it
    ops.check_status(cuda_device)


def test_row_operators_past_32_bit_offsets(cuda_device) -> None:
    """More than 2^31 values: the last rows equal those rows alone, bit for bit."""
    rows, cols, tail = 65600, 32768, 5
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda_device)
    last = _rows(tail, cols, 3).contiguous()
    x[-tail:] = last
    g = _rows(1, cols, 4)[0].contiguous()
    cases = ((ops.quantize_fp8, ()), (ops.silu_and_mul_fp8, ()), (ops.rmsnorm_fp8, (g, 1e-6)),
             (ops.quantize_weight_fp8, ()))
    for op, more in cases:
        own = tail if op is not ops.quantize_weight_fp8 else rows % BLOCK or BLOCK  # the last block of a weight
        q, s = op(x, *more)
        want, scale = op(x[-own:].contiguous(), *more)
        assert torch.equal(q[-own:].view(torch.uint8), want.view(torch.uint8)), op.__name__
        assert torch.equal(s[-scale.shape[0]:], scale), op.__name__
        del q, s
    r = torch.zeros_like(x)
    r[-tail:] = last.flip(0)
    q, s = ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6)
    alone = last.flip(0).contiguous()
    want, scale = ops.fused_add_rmsnorm_fp8(last, alone, g, 1e-6)
    assert torch.equal(q[-tail:].view(torch.uint8), want.view(torch.uint8)) and torch.equal(s[-tail:], scale)
    assert torch.equal(r[-tail:], alone) and not bool(r[:-tail].any())


@pytest.mark.parametrize("rows,n", [(65600, 32768), (16, 100000)])
def test_linear_past_32_bit_offsets(cuda_device, rows: int, n: int) -> None:
    """Outputs (65600 rows) or weight (100000 x 21504) of more than 2^31 values."""
    k = 272 if rows > 16 else 21504
    q, s, wq, ws = _linear_inputs(rows, n, k) if rows > 16 else (*ops.quantize_fp8(_rows(rows, k, 1)), *_wide(n, k))
    y = ops.linear_fp8(q, s, wq, ws)
    ops.check_status(cuda_device)
    t = slice(max(0, rows - 40), rows)
    w, v = wq[-512:], ws[-4:] if n % BLOCK == 0 else None
    if v is None:  # whole blocks of the weight's end
        first = n // BLOCK * BLOCK - 384
        w, v, y = wq[first:], ws[first // BLOCK:], y[:, first:]
    else:
        y = y[:, -512:]
    _linear_check(y[t], q[t], s[t], w, v)


def test_nonfinite_values_show_in_their_rows_only(cuda_device) -> None:
    x = _rows(9, 768, 1).clone()
    x[2, 5], x[4, 300], x[6, 700] = float("nan"), float("inf"), -float("inf")
    q, s = ops.quantize_fp8(x)
    v = _values(q, s)
    for r, c in ((2, 5), (4, 300), (6, 700)):
        assert bool(v[r, c].isnan())
        assert bool(v[r, [j for j in range(768) if j // BLOCK != c // BLOCK]].isfinite().all())
    assert bool(v[[0, 1, 3, 5, 7, 8]].isfinite().all())
    wq, ws = ops.quantize_weight_fp8(_rows(256, 768, 2).contiguous())
    y = ops.linear_fp8(q, s, wq, ws)
    assert bool(y[[2, 4, 6]].isnan().all()) and bool(y[[0, 1, 3, 5, 7, 8]].isfinite().all())
    g = torch.ones(768, dtype=torch.bfloat16, device=cuda_device)
    qn, sn = ops.rmsnorm_fp8(x, g, 1e-6)
    vn = _values(qn, sn)
    assert bool(vn[2].isnan().all()) and bool(vn[4, 300].isnan()) and bool(vn[[0, 1, 3, 5, 7, 8]].isfinite().all())


def test_tiny_values_and_zeros(cuda_device) -> None:
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=cuda_device)
    x[1, 0] = 1e-38  # below the floor of the block maximum: 0 within 2^-10 of the floor's scale
    x[2, 3] = 2.0**-99
    x[3, 130] = 3e38
    q, s = ops.quantize_fp8(x)
    _check_quantised(q, s, x.double(), 2.0**-22)
    assert bool((s[0] == s[1]).all()) and float(s[0, 0]) == pytest.approx(2.0**-100 / 448, rel=2.0**-23)


def test_empty_batch(cuda_device) -> None:
    x = torch.empty(0, 768, dtype=torch.bfloat16, device=cuda_device)
    g = torch.ones(768, dtype=torch.bfloat16, device=cuda_device)
    for q, s in (ops.quantize_fp8(x), ops.rmsnorm_fp8(x, g, 1e-6), ops.fused_add_rmsnorm_fp8(x, x.clone(), g, 1e-6)):
        assert q.shape == (0, 768) and s.shape == (0, 6)
    q, s = ops.silu_and_mul_fp8(x)
    assert q.shape == (0, 384) and s.shape == (0, 3)
    wq, ws = ops.quantize_weight_fp8(_rows(64, 384, 2).contiguous())
    assert ops.linear_fp8(q, s, wq, ws).shape == (0, 64)
    y = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_device)
    assert ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_ADD, residual=y, out=y).shape == (0, 64)


def _mlp(x, r, g, up, down):
    """One MLP of a decoder layer on the 8-bit operators: returns its output, the residual added."""
    q, s = ops.fused_add_rmsnorm_fp8(x, r, g, 1e-6)
    a, sa = ops.silu_and_mul_fp8(ops.linear_fp8(q, s, *up))
    return ops.linear_fp8(a, sa, *down, epilogue=_lib.EPI_ADD, residual=r)


@pytest.mark.parametrize("rows", [1, 8, 13, 200])
def test_mlp_chain_captured_and_on_two_streams(cuda_device, rows: int) -> None:
    """The operators in the order of a decoder layer's MLP: against the same steps in 64
    bits on the quantised operands, replayed from a graph, and two at once."""
    h, f = 768, 2048
    x, r = _rows(rows, h, 1).contiguous(), _rows(rows, h, 2).contiguous()
    g = torch.ones(h, dtype=torch.bfloat16, device=cuda_device)
    up = ops.quantize_weight_fp8((torch.randn(2 * f, h, device=cuda_device) * 0.02).to(torch.bfloat16))
    down = ops.quantize_weight_fp8((torch.randn(h, f, device=cuda_device) * 0.02).to(torch.bfloat16))
    r1 = r.clone()
    want = _mlp(x, r1, g, up, down)
    # each step against 64 bits on the operands that it got
    r2 = r.clone()
    q, s = ops.fused_add_rmsnorm_fp8(x, r2, g, 1e-6)
    gu = ops.linear_fp8(q, s, *up)
    _linear_check(gu, q, s, *up)
    a, sa = ops.silu_and_mul_fp8(gu)
    _check_quantised(a, sa, gu[:, :f].double() * torch.sigmoid(gu[:, :f].double()) * gu[:, f:].double(), 2.0**-16)
    _linear_check(want, a, sa, *down, residual=r2)
    # a captured and replayed chain
    r3 = r.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _mlp(x, r3, g, up, down)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _mlp(x, r3, g, up, down)
    for _ in range(3):
        r3.copy_(r)
        graph.replay()
        assert torch.equal(got, want) and torch.equal(r3, r1)
    # two chains at once, on streams of their own
    streams = [torch.cuda.Stream() for _ in range(2)]
    residuals = [r.clone() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(5):
        outs.clear()
        for st, rr in zip(streams, residuals):
            with torch.cuda.stream(st):
                rr.copy_(r)
                outs.append(_mlp(x, rr, g, up, down))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    ops.check_status(cuda_device)


def test_weight_quantised_just_before_its_linear(cuda_device) -> None:
    """A linear launched right behind the kernel that writes its weight reads the new one."""
    rows, n, k = 8, 4096, 4096
    q, s = ops.quantize_fp8(_rows(rows, k, 4))
    w = [(torch.randn(n, k, device=cuda_device) * 0.02).to(torch.bfloat16) for _ in range(2)]
    want = [ops.linear_fp8(q, s, *ops.quantize_weight_fp8(v)) for v in w]
    wq, ws = ops.quantize_weight_fp8(w[0])
    torch.cuda.synchronize()
    for i in (1, 0, 1, 0):
        _lib.call("aiosb_quantize_weight_fp8", w[i].data_ptr(), n, k, k, wq.data_ptr(), ws.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(ops.linear_fp8(q, s, wq, ws), want[i])


def test_refusals(cuda_device) -> None:
    x = _rows(4, 768, 1).contiguous()
    g = torch.ones(768, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.quantize_fp8(x[:, :24].contiguous())
    with pytest.raises(ValueError, match="16-byte aligned"):
        ops.quantize_fp8(x[:, 4:20])
    with pytest.raises(ValueError, match="row stride"):
        ops.quantize_fp8(x[:1].expand(4, -1))
    with pytest.raises(ValueError, match="contiguous"):
        ops.quantize_fp8(x.t())
    with pytest.raises(ValueError, match="bfloat16"):
        ops.quantize_fp8(x.float())
    with pytest.raises(ValueError, match="at most 32768"):
        ops.rmsnorm_fp8(torch.zeros(1, 32784, dtype=torch.bfloat16, device=cuda_device),
                        torch.ones(32784, dtype=torch.bfloat16, device=cuda_device), 1e-6)
    with pytest.raises(ValueError, match="weight"):
        ops.rmsnorm_fp8(x, g[:760], 1e-6)
    with pytest.raises(ValueError, match="residual"):
        ops.fused_add_rmsnorm_fp8(x, x[:3], g, 1e-6)
    q, s = ops.quantize_fp8(x)
    wq, ws = ops.quantize_weight_fp8(_rows(64, 768, 2).contiguous())
    with pytest.raises(ValueError, match="x_scale"):
        ops.linear_fp8(q, s[:3], wq, ws)
    with pytest.raises(ValueError, match="weight_scale"):
        ops.linear_fp8(q, s, wq, ws.repeat(2, 1))
    with pytest.raises(ValueError, match="expects x"):
        ops.linear_fp8(q, s, wq[:, :752], ws)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.linear_fp8(q, s, wq[:60], ws)
    with pytest.raises(ValueError, match="residual"):
        ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_ADD)
    with pytest.raises(ValueError, match="unknown epilogue"):
        ops.linear_fp8(q, s, wq, ws, epilogue=_lib.EPI_SILU_MUL)
    with pytest.raises(ValueError, match="output"):
        ops.linear_fp8(q, s, wq, ws, out=torch.empty(4, 64, device=cuda_device))
