"""Argument checks of the 8-bit linear entry points: they run before any CUDA call, so
every refusal is seen on a CPU machine."""

from __future__ import annotations

import pytest
import torch

from aios_b200 import _lib
from aios_b200.kernel import ops

P = 1 << 20  # an aligned address that is never read: every call below is refused first


def _refused(name: str, args: list, code: int, text: str) -> None:
    rc = getattr(_lib.load(), name)(*args)
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


ROWS = {
    "aiosb_quantize_fp8": [P, 4, 256, 256, P, P, None],
    "aiosb_quantize_weight_fp8": [P, 4, 256, 256, P, P, None],
    "aiosb_silu_mul_fp8": [P, 4, 256, 512, P, P, None],
    "aiosb_rmsnorm_fp8": [P, 4, 256, 256, None, None, P, 1e-6, P, P, None],
}


@pytest.mark.parametrize("name", list(ROWS))
def test_row_operators_refuse(name: str) -> None:
    q, scale = (8, 9) if "rmsnorm" in name else (4, 5)

    def with_(**changes):
        a = list(ROWS[name])
        for i, v in changes.items():
            a[int(i[1:])] = v
        return a

    inv, uns, mis = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_MISALIGNED
    _refused(name, with_(_1=-1), inv, "bad sizes")
    _refused(name, with_(_2=0), inv, "bad sizes")
    _refused(name, with_(_2=248), uns, "multiple of 16")
    _refused(name, with_(_1=1 << 31), uns, "too many")
    _refused(name, with_(_3=248), inv, "row stride")
    _refused(name, with_(_3=516), inv, "row stride")
    _refused(name, with_(_0=None), inv, "null")
    _refused(name, with_(**{f"_{scale}": None}), inv, "null")
    _refused(name, with_(_0=P + 2), mis, "aligned")
    _refused(name, with_(**{f"_{q}": P + 8}), mis, "aligned")
    assert getattr(_lib.load(), name)(*with_(_1=0, _0=None)) == _lib.OK  # nothing to do


def test_norm_refuses() -> None:
    a = ROWS["aiosb_rmsnorm_fp8"]
    _refused("aiosb_rmsnorm_fp8", [P, 4, 32784, 32784, *a[4:]], _lib.ERR_UNSUPPORTED, "at most 32768")
    _refused("aiosb_rmsnorm_fp8", [*a[:4], P, None, *a[6:]], _lib.ERR_INVALID_ARG, "go together")
    _refused("aiosb_rmsnorm_fp8", [*a[:6], P + 4, *a[7:]], _lib.ERR_MISALIGNED, "weight and residual")
    _refused("aiosb_rmsnorm_fp8", [*a[:4], P + 4, P, *a[6:]], _lib.ERR_MISALIGNED, "weight and residual")


def test_linear_refuses() -> None:
    good = dict(x=P, xs=256, sx=P, rows=4, k=256, w=P, sw=P, n=64, y=P, ys=64, epi=0, res=None, rs=0, status=None,
                stream=None)

    def call(code, text, **changes):
        _refused("aiosb_linear_fp8", list({**good, **changes}.values()), code, text)

    inv, uns, mis = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_MISALIGNED
    call(inv, "bad sizes", rows=-1)
    call(inv, "bad sizes", k=0)
    call(uns, "multiple of 8", n=60)
    call(uns, "multiple of 16", k=248)
    call(uns, "too large", rows=1 << 31)
    call(inv, "unknown epilogue", epi=_lib.EPI_SILU_MUL)
    call(inv, "needs an aligned residual", epi=_lib.EPI_ADD)
    call(inv, "needs an aligned residual", epi=_lib.EPI_ADD, res=P + 8, rs=64)
    call(inv, "needs an aligned residual", epi=_lib.EPI_ADD, res=P, rs=56)
    call(inv, "x row stride", xs=240)
    call(inv, "x row stride", xs=264)
    call(inv, "y row stride", ys=56)
    call(inv, "y row stride", ys=68)
    call(inv, "null", sx=None)
    call(inv, "null", y=None)
    call(mis, "aligned", x=P + 8)
    call(mis, "aligned", w=P + 8)
    assert _lib.load().aiosb_linear_fp8(*{**good, "rows": 0, "x": None, "y": None}.values()) == _lib.OK


def test_wrappers_want_cuda_tensors() -> None:
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.quantize_weight_fp8(x), lambda: ops.silu_and_mul_fp8(x),
                 lambda: ops.rmsnorm_fp8(x, x[0], 1e-6), lambda: ops.fused_add_rmsnorm_fp8(x, x, x[0], 1e-6),
                 lambda: ops.linear_fp8(x.to(torch.float8_e4m3fn), x, x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
