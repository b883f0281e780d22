"""Torch-tensor wrappers over the C ABI (``aios_b200._lib``).

Each wrapper validates shapes/dtypes on the host, passes raw device addresses and
the current CUDA stream, and never computes anything itself: every op here runs
as a hand-written sm_100a kernel. Device-side errors land in a per-device int32
status word that :func:`check_status` turns into a ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext

import torch

from .. import _lib

_STATUS: dict[int, torch.Tensor] = {}

# Bytes the host side stages to / from the device outside the runtime's own
# counters (prefill ids, attention metadata); read by the benchmark.
transfer_bytes = {"h2d": 0, "d2h": 0}


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def status_word(device: torch.device) -> torch.Tensor:
    """The per-device int32 status word that kernels report device faults into."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    st = _STATUS.get(index)
    if st is None:
        st = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        _STATUS[index] = st
    return st


def _status_pointer(index: int) -> int:
    st = _STATUS.get(index)
    return (st if st is not None else status_word(torch.device("cuda", index))).data_ptr()


def check_status(device: torch.device, reset: bool = True) -> None:
    """Raises if any kernel on `device` reported a device-side fault (syncs)."""
    st = status_word(device)
    code = int(st.item())
    if code:
        if reset:
            st.zero_()
        raise RuntimeError(f"aios_b200 device status {code}: {_lib.DEVICE_STATUS_NAMES.get(code, 'unknown')}")


def host_device_pointer(pinned: torch.Tensor) -> int:
    """Device address of a page-locked host tensor (for host-mapped flags)."""
    if not pinned.is_pinned():
        raise ValueError("host_device_pointer needs a pinned CPU tensor")
    out = ctypes.c_void_p()
    _lib.call("aiosb_host_device_pointer", pinned.data_ptr(), ctypes.byref(out))
    return int(out.value)


def _require_cuda(*tensors: torch.Tensor, what: str) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError(f"{what} requires CUDA tensors")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# KV store (aios/kernel/store.py:32-61)
# ---------------------------------------------------------------------------
def store_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    indices: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
) -> None:
    """Scatter a flat batch of K/V vectors into a contiguous CUDA cache."""
    if k_cache.ndim != 3 or v_cache.ndim != 3:
        raise ValueError("KV cache must have shape (num_slots, num_heads, head_dim)")
    if k.shape[1:] != k_cache.shape[1:] or v.shape[1:] != v_cache.shape[1:]:
        raise ValueError("K/V input shape does not match the cache layout")
    if indices.numel() != k.shape[0] or k.shape != v.shape:
        raise ValueError("KV write indices and K/V tensors must have matching token counts")
    _require_cuda(k_cache, v_cache, indices, k, v, what="store_cache")
    if k.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("store_cache expects bf16 K/V and cache")
    for name, t in (("k", k), ("v", v)):
        if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
            raise ValueError(f"{name} rows must be contiguous within a token")
    if not (k_cache[0].is_contiguous() and v_cache[0].is_contiguous()):
        raise ValueError("KV cache rows must be contiguous")
    idx = indices.to(torch.int32).contiguous()
    width = k_cache.shape[1] * k_cache.shape[2]
    _lib.call(
        "aiosb_kv_store",
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        k_cache.stride(0),
        k_cache.shape[0],
        idx.data_ptr(),
        k.shape[0],
        k.data_ptr(),
        k.stride(0),
        v.data_ptr(),
        v.stride(0),
        width,
        status_word(k.device).data_ptr(),
        _stream(k.device),
    )


# ---------------------------------------------------------------------------
# AttnRes mixer (aios/kernel/attnres.py:130-223)
# ---------------------------------------------------------------------------
def b200_attnres_mix(
    bank: torch.Tensor,
    partial: torch.Tensor | None,
    weighted_query: torch.Tensor,
    eps: float,
    *,
    score_buffer: torch.Tensor | None = None,
    output_buffer: torch.Tensor | None = None,
) -> torch.Tensor:
    """FP32 depth routing and BF16 value aggregation in one sm_100a kernel.

    Same signature and layout checks as the reference ``triton_attnres_mix``;
    ``score_buffer`` is accepted and validated but unused, because the fused
    kernel keeps the [S, N] scores in registers.
    """
    if not bank.is_cuda:
        raise ValueError("B200 AttnRes requires CUDA tensors")
    if bank.ndim != 3:
        raise ValueError("bank must have shape [S,N,D]")
    if not bank.is_contiguous():
        raise ValueError("bank must be contiguous for the B200 pointer layout")
    bank_sources, num_tokens, hidden_size = bank.shape
    if bank_sources < 1 or num_tokens < 1 or hidden_size < 1:
        raise ValueError("bank dimensions must be positive")
    total_sources = bank_sources + int(partial is not None)
    if partial is not None and partial.shape != bank.shape[1:]:
        raise ValueError("partial must match bank [N,D]")
    if partial is not None and not partial.is_contiguous():
        raise ValueError("partial must be contiguous")
    if weighted_query.shape != (hidden_size,):
        raise ValueError("weighted_query must match hidden size")
    if not weighted_query.is_contiguous():
        raise ValueError("weighted_query must be contiguous")
    if weighted_query.dtype != torch.float32:
        raise ValueError("weighted_query must be float32")
    if bank.dtype != torch.bfloat16 or (partial is not None and partial.dtype != torch.bfloat16):
        raise ValueError("B200 AttnRes expects bf16 bank/partial")
    if score_buffer is not None:
        if score_buffer.dtype != torch.float32 or score_buffer.device != bank.device:
            raise ValueError("score_buffer must be CUDA float32 on bank device")
        if (
            score_buffer.shape[0] < total_sources
            or score_buffer.shape[1] != num_tokens
            or not score_buffer.is_contiguous()
        ):
            raise ValueError("score_buffer must be contiguous [capacity_sources, num_tokens]")
    if output_buffer is None:
        output = torch.empty_like(bank[0])
    else:
        if output_buffer.shape != bank.shape[1:]:
            raise ValueError("output_buffer must match bank [N,D]")
        if output_buffer.dtype != bank.dtype or output_buffer.device != bank.device:
            raise ValueError("output_buffer must match bank dtype/device")
        if not output_buffer.is_contiguous():
            raise ValueError("output_buffer must be contiguous")
        output = output_buffer
    _lib.call(
        "aiosb_attnres_mix",
        bank.data_ptr(),
        bank_sources,
        num_tokens,
        hidden_size,
        _ptr(partial),
        weighted_query.data_ptr(),
        float(eps),
        output.data_ptr(),
        status_word(bank.device).data_ptr(),
        _stream(bank.device),
    )
    return output


def b200_attnres_mix_rmsnorm(
    bank: torch.Tensor,
    partial: torch.Tensor | None,
    weighted_query: torch.Tensor,
    eps: float,
    norm_weight: torch.Tensor,
    norm_eps: float,
    *,
    output_buffer: torch.Tensor | None = None,
    stable_sources: int = 0,
) -> torch.Tensor:
    """rmsnorm(b200_attnres_mix(bank, partial, weighted_query, eps)) * norm_weight
    in one kernel: the mixer and the RMSNorm that consumes its output in the Block
    AttnRes layers. The mixer result itself is not returned. ``stable_sources``:
    the first bank sources were written before the previous kernel on the stream
    began, so the kernel may read them before waiting on it."""
    if not (bank.is_cuda and bank.dtype == torch.bfloat16 and bank.ndim == 3 and bank.is_contiguous()):
        raise ValueError("bank must be a contiguous CUDA bf16 [S,N,D] tensor")
    sources, tokens, hidden = bank.shape
    if partial is not None and (partial.shape != bank.shape[1:] or not partial.is_contiguous()
                                or partial.dtype != torch.bfloat16):
        raise ValueError("partial must be a contiguous bf16 [N,D] tensor matching bank")
    if weighted_query.shape != (hidden,) or weighted_query.dtype != torch.float32:
        raise ValueError("weighted_query must be float32 [D]")
    if norm_weight.shape != (hidden,) or norm_weight.dtype != torch.bfloat16 or not norm_weight.is_contiguous():
        raise ValueError("norm_weight must be a contiguous bf16 [D] tensor")
    output = torch.empty_like(bank[0]) if output_buffer is None else output_buffer
    if output.shape != bank.shape[1:] or not output.is_contiguous():
        raise ValueError("output_buffer must be a contiguous [N,D] tensor")
    _lib.call(
        "aiosb_attnres_mix_rmsnorm",
        bank.data_ptr(), sources, tokens, hidden, _ptr(partial), weighted_query.contiguous().data_ptr(), float(eps),
        norm_weight.data_ptr(), float(norm_eps), int(stable_sources), output.data_ptr(), _stream(bank.device),
    )
    return output


MIX_MAX_SOURCES = 10  # aiosb_linear_attnres_rmsnorm: bank + partial
MIX_MAX_ROWS = 8


def linear_attnres_rmsnorm_eligible(bank: torch.Tensor, partial: torch.Tensor | None, stable: int) -> bool:
    sources, tokens, hidden = bank.shape
    late = sources - stable + (partial is not None)
    return (tokens <= MIX_MAX_ROWS and hidden == 768 and 0 <= stable <= sources and late <= 2
            and sources + (partial is not None) <= MIX_MAX_SOURCES)


def linear_attnres_rmsnorm(
    bank: torch.Tensor,
    partial: torch.Tensor | None,
    stable_sources: int,
    weighted_query: torch.Tensor,
    mix_eps: float,
    norm_weight: torch.Tensor,
    norm_eps: float,
    weight: torch.Tensor,
    *,
    epilogue: int = _lib.EPI_STORE,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``linear(rmsnorm(attnres_mix(bank, partial)) * norm_weight, weight)`` in one
    decode kernel (at most 8 tokens, hidden 768): the mixer's rows are built inside
    the linear. The first ``stable_sources`` bank sources were written before the
    previous kernel on the stream began."""
    if not linear_attnres_rmsnorm_eligible(bank, partial, stable_sources):
        raise ValueError("linear_attnres_rmsnorm: 1..8 tokens, hidden 768, <= 10 sources, <= 2 read late")
    _require_cuda(bank, weighted_query, norm_weight, weight, what="linear_attnres_rmsnorm")
    sources, tokens, hidden = bank.shape
    n = weight.shape[0]
    cols = n // 2 if epilogue == _lib.EPI_SILU_MUL else n
    if out is None:
        out = torch.empty((tokens, cols), dtype=bank.dtype, device=bank.device)
    _lib.call(
        "aiosb_linear_attnres_rmsnorm", bank.data_ptr(), sources, int(stable_sources), tokens, _ptr(partial),
        weighted_query.contiguous().data_ptr(), float(mix_eps), norm_weight.data_ptr(), float(norm_eps),
        weight.data_ptr(), n, hidden, out.data_ptr(), out.stride(0), epilogue, status_word(bank.device).data_ptr(),
        _stream(bank.device),
    )
    return out


# ---------------------------------------------------------------------------
# Norms / activations / embedding (aios/layers/{norm,activation,embedding}.py)
# ---------------------------------------------------------------------------
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm over the last dim of a 2-D [T, H] or 3-D [T, heads, d] view."""
    _require_cuda(x, weight, what="rmsnorm")
    if out is None:
        out = torch.empty_like(x)
    if x.ndim == 2:
        x3, o3 = x.unsqueeze(1), out.unsqueeze(1)
    elif x.ndim == 3:
        x3, o3 = x, out
    else:
        raise ValueError("rmsnorm expects a 2-D or 3-D tensor")
    hidden = x3.shape[2]
    if weight.shape != (hidden,):
        raise ValueError("rmsnorm weight must match the last dimension")
    for t in (x3, o3):
        if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != hidden):
            raise ValueError("rmsnorm rows must be dense within a token")
    _lib.call(
        "aiosb_rmsnorm",
        x3.data_ptr(),
        x3.shape[0] * x3.shape[1],
        hidden,
        x3.shape[1],
        x3.stride(0),
        weight.data_ptr(),
        float(eps),
        o3.data_ptr(),
        o3.stride(0),
        _stream(x.device),
    )
    return out


def fused_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float) -> None:
    """residual += x; x = rmsnorm(residual) (in place, FlashInfer semantics)."""
    _require_cuda(x, residual, weight, what="fused_add_rmsnorm")
    if x.shape != residual.shape or x.ndim != 2 or not x.is_contiguous() or not residual.is_contiguous():
        raise ValueError("fused_add_rmsnorm expects matching contiguous [T, H] tensors")
    _lib.call(
        "aiosb_add_rmsnorm",
        x.data_ptr(),
        residual.data_ptr(),
        x.shape[0],
        x.shape[1],
        weight.data_ptr(),
        float(eps),
        _stream(x.device),
    )


def silu_and_mul(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_cuda(x, what="silu_and_mul")
    if x.ndim != 2 or x.shape[1] % 2 or not x.is_contiguous():
        raise ValueError("silu_and_mul expects a contiguous [T, 2F] tensor")
    f = x.shape[1] // 2
    if out is None:
        out = torch.empty((x.shape[0], f), dtype=x.dtype, device=x.device)
    _lib.call("aiosb_silu_mul", x.data_ptr(), x.shape[0], f, out.data_ptr(), _stream(x.device))
    return out


def embedding(ids: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_cuda(ids, weight, what="embedding")
    ids = ids.contiguous()
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("embedding ids must be int32 or int64")
    if out is None:
        out = torch.empty((ids.numel(), weight.shape[1]), dtype=weight.dtype, device=weight.device)
    _lib.call(
        "aiosb_embedding",
        ids.data_ptr(),
        int(ids.dtype == torch.int64),
        ids.numel(),
        weight.data_ptr(),
        weight.shape[0],
        weight.shape[1],
        out.data_ptr(),
        status_word(ids.device).data_ptr(),
        _stream(ids.device),
    )
    return out


# ---------------------------------------------------------------------------
# Linear (tcgen05 GEMM)
# ---------------------------------------------------------------------------
def linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    out: torch.Tensor | None = None,
    epilogue: int = _lib.EPI_STORE,
    residual: torch.Tensor | None = None,
    tile_stats: torch.Tensor | None = None,
    early_dependents: bool = False,
) -> torch.Tensor:
    """y = x @ weight.T on the tensor cores (bf16 in, fp32 accumulate, bf16 out).

    ``epilogue=EPI_ADD`` returns ``residual + bf16(x @ weight.T)`` (residual may
    be ``out`` for an in-place add). ``tile_stats`` and ``early_dependents`` as in
    ``linear_stat_norm``."""
    _require_cuda(x, weight, what="linear")
    if x.ndim != 2 or weight.ndim != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError("linear expects x [T, K] and weight [N, K]")
    if not x.is_contiguous() or not weight.is_contiguous():
        raise ValueError("linear expects contiguous x and weight")
    n = weight.shape[0]
    cols = n // 2 if epilogue == _lib.EPI_SILU_MUL else n
    if epilogue == _lib.EPI_ADD:
        if residual is None or residual.shape != (x.shape[0], n) or residual.stride(1) != 1:
            raise ValueError("the add epilogue needs a residual [rows, n] with contiguous rows")
    if out is None:
        out = torch.empty((x.shape[0], cols), dtype=x.dtype, device=x.device)
    if out.stride(1) != 1:
        raise ValueError("linear output rows must be contiguous")
    if tile_stats is not None:
        _check_tile_stats(tile_stats, epilogue, x.shape[0], x.shape[1], n)
        _lib.call("aiosb_linear_tiles", x.data_ptr(), x.shape[0], x.shape[1], weight.data_ptr(), n, out.data_ptr(),
                  out.stride(0), tile_stats.data_ptr(), status_word(x.device).data_ptr(), _stream(x.device))
        return out
    _lib.call(
        "aiosb_linear",
        x.data_ptr(),
        x.shape[0],
        x.shape[1],
        weight.data_ptr(),
        n,
        out.data_ptr(),
        out.stride(0),
        epilogue | (_lib.LINEAR_EARLY_DEPENDENTS if early_dependents else 0),
        _ptr(residual) if epilogue == _lib.EPI_ADD else None,
        residual.stride(0) if (epilogue == _lib.EPI_ADD and residual is not None) else 0,
        status_word(x.device).data_ptr(),
        _stream(x.device),
    )
    return out


MAX_NORM_ROWS = 64  # rows the fused-RMSNorm GEMM prologue handles


def linear_rmsnorm(
    x: torch.Tensor,
    residual_in: torch.Tensor | None,
    norm_weight: torch.Tensor,
    eps: float,
    weight: torch.Tensor,
    *,
    residual_out: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    epilogue: int = _lib.EPI_STORE,
) -> torch.Tensor:
    """``linear(rmsnorm(x + residual_in) * norm_weight, weight)`` in one kernel
    (rows <= 64); ``residual_out`` receives ``x + residual_in`` when given."""
    _require_cuda(x, norm_weight, weight, what="linear_rmsnorm")
    rows, k = x.shape
    if rows > MAX_NORM_ROWS:
        raise ValueError(f"linear_rmsnorm handles at most {MAX_NORM_ROWS} rows")
    for t in (x, residual_in, residual_out):
        if t is not None and (t.shape != (rows, k) or not t.is_contiguous()):
            raise ValueError("linear_rmsnorm expects contiguous [rows, k] x / residual tensors")
    n = weight.shape[0]
    cols = n // 2 if epilogue == _lib.EPI_SILU_MUL else n
    if out is None:
        out = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    _lib.call(
        "aiosb_linear_rmsnorm",
        x.data_ptr(),
        _ptr(residual_in),
        _ptr(residual_out),
        norm_weight.data_ptr(),
        float(eps),
        rows,
        k,
        weight.data_ptr(),
        n,
        out.data_ptr(),
        out.stride(0),
        epilogue,
        None,
        0,
        status_word(x.device).data_ptr(),
        _stream(x.device),
    )
    return out


class RowStats:
    """RMSNorm statistics of a residual stream handed from one GEMM to the next:
    ``x`` [T, D] fp32 (the un-rounded residual sum) and ``ss`` [parts, T] fp32
    (sums of squares over each 128-column tile, or over the whole row)."""

    __slots__ = ("x", "ss")

    def __init__(self, x: torch.Tensor, ss: torch.Tensor):
        self.x, self.ss = x, ss

    @classmethod
    def empty(cls, rows: int, hidden: int, parts: int, device: torch.device) -> "RowStats":
        return cls(torch.empty((rows, hidden), dtype=torch.float32, device=device),
                   torch.empty((parts, rows), dtype=torch.float32, device=device))

    @property
    def parts(self) -> int:
        return self.ss.shape[0]

    def rows(self, start: int, stop: int) -> "RowStats":
        return RowStats(self.x[start:stop], self.ss[:, start:stop])

    def select(self, idx: torch.Tensor) -> "RowStats":
        return RowStats(self.x.index_select(0, idx).contiguous(), self.ss.index_select(1, idx).contiguous())


def embedding_stat(ids: torch.Tensor, weight: torch.Tensor) -> tuple[torch.Tensor, RowStats]:
    """Embedding rows plus their RMSNorm statistics (one part per row)."""
    _require_cuda(ids, weight, what="embedding_stat")
    ids = ids.contiguous()
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("embedding ids must be int32 or int64")
    t, d = ids.numel(), weight.shape[1]
    out = torch.empty((t, d), dtype=weight.dtype, device=weight.device)
    st = RowStats.empty(t, d, 1, weight.device)
    _lib.call("aiosb_embedding_stat", ids.data_ptr(), int(ids.dtype == torch.int64), t, weight.data_ptr(),
              weight.shape[0], d, out.data_ptr(), st.x.data_ptr(), st.ss.data_ptr(),
              status_word(ids.device).data_ptr(), _stream(ids.device))
    return out, st


def linear_add_stat(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor) -> RowStats:
    """residual <- bf16(residual + bf16(x @ weight.T)) in place, returning the
    RMSNorm statistics of the new residual stream."""
    _require_cuda(x, weight, residual, what="linear_add_stat")
    if x.ndim != 2 or weight.ndim != 2 or x.shape[1] != weight.shape[1] or not x.is_contiguous():
        raise ValueError("linear_add_stat expects contiguous x [T, K] and weight [N, K]")
    rows, n = x.shape[0], weight.shape[0]
    if residual.shape != (rows, n) or residual.stride(1) != 1:
        raise ValueError("linear_add_stat needs a residual [rows, n] with contiguous rows")
    st = RowStats.empty(rows, n, n // 8, x.device)
    parts = ctypes.c_int64(0)
    _lib.call("aiosb_linear_add_stat", x.data_ptr(), rows, x.shape[1], weight.data_ptr(), n, residual.data_ptr(),
              residual.stride(0), residual.data_ptr(), residual.stride(0), st.x.data_ptr(), st.ss.data_ptr(),
              st.ss.stride(0), ctypes.byref(parts), status_word(x.device).data_ptr(), _stream(x.device))
    return RowStats(st.x, st.ss[: parts.value])


def linear_stat_norm(
    stats: RowStats,
    norm_weight: torch.Tensor,
    eps: float,
    weight: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    epilogue: int = _lib.EPI_STORE,
    tile_stats: torch.Tensor | None = None,
    early_dependents: bool = False,
) -> torch.Tensor:
    """``linear(rmsnorm(s) * norm_weight, weight)`` with s and its sums of squares
    from ``stats``; the normalised rows exist only inside the GEMM.
    ``early_dependents``: the next kernel may launch before this one's wait
    (``LINEAR_EARLY_DEPENDENTS``; the caller vouches for the successor). With
    ``tile_stats`` (fp32, [n / 16, rows, 4], see ``tile_stats_eligible``) the
    store epilogue also writes each 16-column tile's (max, sum of exp(v - max),
    min, NaN flag) of the stored values."""
    _require_cuda(stats.x, norm_weight, weight, what="linear_stat_norm")
    rows, k = stats.x.shape
    if weight.shape[1] != k or stats.x.stride(1) != 1 or stats.x.stride(0) != k or stats.ss.stride(1) != 1:
        raise ValueError("linear_stat_norm expects contiguous statistics [rows, k] matching the weight")
    n = weight.shape[0]
    cols = n // 2 if epilogue == _lib.EPI_SILU_MUL else n
    if out is None:
        out = torch.empty((rows, cols), dtype=weight.dtype, device=weight.device)
    if tile_stats is not None:
        _check_tile_stats(tile_stats, epilogue, rows, k, n)
        _lib.call("aiosb_linear_stat_norm_tiles", stats.x.data_ptr(), stats.ss.data_ptr(), stats.ss.stride(0),
                  stats.parts, norm_weight.data_ptr(), float(eps), rows, k, weight.data_ptr(), n, out.data_ptr(),
                  out.stride(0), tile_stats.data_ptr(), status_word(weight.device).data_ptr(),
                  _stream(weight.device))
        return out
    flags = _lib.LINEAR_EARLY_DEPENDENTS if early_dependents else 0
    _lib.call("aiosb_linear_stat_norm", stats.x.data_ptr(), stats.ss.data_ptr(), stats.ss.stride(0), stats.parts,
              norm_weight.data_ptr(), float(eps), rows, k, weight.data_ptr(), n, out.data_ptr(), out.stride(0),
              epilogue | flags, None, 0, status_word(weight.device).data_ptr(), _stream(weight.device))
    return out


def _check_tile_stats(tile_stats: torch.Tensor, epilogue: int, rows: int, k: int, n: int) -> None:
    if epilogue != _lib.EPI_STORE or not tile_stats_eligible(rows, k, n):
        raise ValueError("tile statistics need the store epilogue, rows <= 16, k <= 768, n % 16 == 0")
    if tile_stats.dtype != torch.float32 or not tile_stats.is_contiguous() or tile_stats.numel() < n // 16 * rows * 4:
        raise ValueError("tile_stats must be contiguous fp32 with n / 16 * rows * 4 elements")


def tile_stats_eligible(rows: int, k: int, n: int) -> bool:
    """Whether ``linear_stat_norm`` can write tile statistics for this shape (the
    library's answer: the register-operand path with rows <= 16, k a multiple of
    256 up to 768, n % 16 == 0)."""
    return bool(_lib.load().aiosb_linear_tile_stats_eligible(rows, k, n))


def pack_gate_up(weight: torch.Tensor) -> torch.Tensor:
    """[gate | up] rows ([2F, K]) -> 64-row interleaved blocks for EPI_SILU_MUL."""
    two_f, k = weight.shape
    f = two_f // 2
    if f % 64:
        raise ValueError("gate/up width must be a multiple of 64")
    gate = weight[:f].reshape(f // 64, 64, k)
    up = weight[f:].reshape(f // 64, 64, k)
    return torch.stack((gate, up), dim=1).reshape(two_f, k).contiguous()


# ---------------------------------------------------------------------------
# 8-bit linears: e4m3 values, one fp32 scale for each block of 128
# ---------------------------------------------------------------------------
FP8_BLOCK = 128
FP8_DTYPE = torch.float8_e4m3fn


def _launch(index: int, name: str, *args) -> None:
    """Calls a launching entry point on the current stream of device `index` (its last
    argument), with that device current."""
    if index == torch._C._cuda_getDevice():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


# These wrappers run in about the time of one small launch, so their checks are spelled
# out on plain attributes and outputs come from the allocator's shortest entry: a decode
# step is bound by the host's launch rate otherwise.
_new_cuda = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)


def _empty_vector(x: torch.Tensor, size: int, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised [size] tensor on x's device."""
    if _new_cuda is not None and x.get_device() == torch._C._cuda_getDevice():
        return _new_cuda((size,), (1,), dtype)
    return x.new_empty(size, dtype=dtype)


def _empty_rows(x: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised contiguous [rows, cols] tensor on x's device."""
    if _new_cuda is not None and x.get_device() == torch._C._cuda_getDevice():
        return _new_cuda((rows, cols), (cols, 1), dtype)
    return x.new_empty(rows, cols, dtype=dtype)


def _check_rows(what: str, x: torch.Tensor, dtype: torch.dtype) -> tuple[int, int, int]:
    """`x` as rows with contiguous columns on a CUDA device: (rows, cols, row stride)."""
    if x.dtype is dtype and x.ndim == 2 and x.is_cuda:
        rows, cols = x.shape
        if x.is_contiguous():
            return rows, cols, cols
        stride, inner = x.stride()
        if inner == 1 or cols == 1:
            return rows, cols, stride if rows > 1 else cols
        raise ValueError(f"{what} rows must be contiguous")
    if not x.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    raise ValueError(f"{what} expects a 2-D {dtype} tensor")


def _check_dense(what: str, name: str, t: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype,
                 index: int) -> None:
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor of shape {list(shape)} on cuda:{index}")


def _fp8_outputs(what: str, x: torch.Tensor, rows: int, cols: int, out: torch.Tensor | None,
                 scale: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    if out is None:
        out = _empty_rows(x, rows, cols, FP8_DTYPE)
    else:
        _check_dense(what, "out", out, (rows, cols), FP8_DTYPE, x.get_device())
    if scale is None:
        scale = _empty_rows(x, rows, -(-cols // FP8_BLOCK), torch.float32)
    else:
        _check_dense(what, "scale", scale, (rows, -(-cols // FP8_BLOCK)), torch.float32, x.get_device())
    return out, scale


def quantize_fp8(x: torch.Tensor, *, out: torch.Tensor | None = None,
                 scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 rows [T, H] to (e4m3 [T, H], scale [T, ceil(H / 128)]): a scale for each 128
    columns of a row, ``x ~ q * scale``. H is a multiple of 16; rows may be strided."""
    rows, cols, stride = _check_rows("quantize_fp8", x, torch.bfloat16)
    out, scale = _fp8_outputs("quantize_fp8", x, rows, cols, out, scale)
    _launch(x.get_device(), "aiosb_quantize_fp8", x.data_ptr(), rows, cols, stride, out.data_ptr(), scale.data_ptr())
    return out, scale


def quantize_weight_fp8(weight: torch.Tensor, *, out: torch.Tensor | None = None,
                        scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """A bf16 weight [N, K] to (e4m3 [N, K], scale [ceil(N / 128), ceil(K / 128)]): a scale
    for each 128 x 128 block. K is a multiple of 16; rows may be strided."""
    n, k, stride = _check_rows("quantize_weight_fp8", weight, torch.bfloat16)
    tall, wide = -(-n // FP8_BLOCK), -(-k // FP8_BLOCK)
    if out is None:
        out = _empty_rows(weight, n, k, FP8_DTYPE)
    else:
        _check_dense("quantize_weight_fp8", "out", out, (n, k), FP8_DTYPE, weight.get_device())
    if scale is None:
        scale = _empty_rows(weight, tall, wide, torch.float32)
    else:
        _check_dense("quantize_weight_fp8", "scale", scale, (tall, wide), torch.float32, weight.get_device())
    _launch(weight.get_device(), "aiosb_quantize_weight_fp8", weight.data_ptr(), n, k, stride, out.data_ptr(),
            scale.data_ptr())
    return out, scale


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float, *, out: torch.Tensor | None = None,
                scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8(rmsnorm(x, weight, eps))`` in one kernel, without the bf16 rounding
    between the two. x is [T, H] with H a multiple of 16, at most 32768."""
    rows, hidden, stride = _check_rows("rmsnorm_fp8", x, torch.bfloat16)
    index = x.get_device()
    _check_dense("rmsnorm_fp8", "weight", weight, (hidden,), torch.bfloat16, index)
    out, scale = _fp8_outputs("rmsnorm_fp8", x, rows, hidden, out, scale)
    _launch(index, "aiosb_rmsnorm_fp8", x.data_ptr(), rows, hidden, stride, None, None, weight.data_ptr(), float(eps),
            out.data_ptr(), scale.data_ptr())
    return out, scale


def fused_add_rmsnorm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *,
                          residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
                          scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``fused_add_rmsnorm`` with 8-bit output: residual += x (in place, or into
    ``residual_out``), and the quantised rmsnorm of the fp32 sum is returned; x is kept."""
    rows, hidden, stride = _check_rows("fused_add_rmsnorm_fp8", x, torch.bfloat16)
    index = x.get_device()
    _check_dense("fused_add_rmsnorm_fp8", "weight", weight, (hidden,), torch.bfloat16, index)
    _check_dense("fused_add_rmsnorm_fp8", "residual", residual, (rows, hidden), torch.bfloat16, index)
    if residual_out is None:
        residual_out = residual
    else:
        _check_dense("fused_add_rmsnorm_fp8", "residual_out", residual_out, (rows, hidden), torch.bfloat16, index)
    out, scale = _fp8_outputs("fused_add_rmsnorm_fp8", x, rows, hidden, out, scale)
    if rows:
        _launch(index, "aiosb_rmsnorm_fp8", x.data_ptr(), rows, hidden, stride, residual.data_ptr(),
                residual_out.data_ptr(), weight.data_ptr(), float(eps), out.data_ptr(), scale.data_ptr())
    return out, scale


def silu_and_mul_fp8(x: torch.Tensor, *, out: torch.Tensor | None = None,
                     scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8(silu_and_mul(x))`` in one kernel, without the bf16 rounding between
    the two: x is [T, 2F] ([gate | up]) with F a multiple of 16."""
    rows, width, stride = _check_rows("silu_and_mul_fp8", x, torch.bfloat16)
    if width % 2:
        raise ValueError("silu_and_mul_fp8 expects a [T, 2F] tensor")
    f = width // 2
    out, scale = _fp8_outputs("silu_and_mul_fp8", x, rows, f, out, scale)
    _launch(x.get_device(), "aiosb_silu_mul_fp8", x.data_ptr(), rows, f, stride, out.data_ptr(), scale.data_ptr())
    return out, scale


def linear_fp8(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    epilogue: int = _lib.EPI_STORE,
    residual: torch.Tensor | None = None,
    stable_weight: bool = False,
) -> torch.Tensor:
    """y = x @ weight.T of quantised rows [T, K] and weight [N, K] (``quantize_fp8``,
    ``quantize_weight_fp8``) on the 8-bit tensor cores, fp32 sums, bf16 out.

    ``epilogue=EPI_ADD`` returns ``residual + x @ weight.T`` with one rounding (residual
    may be ``out`` for an in-place add). N is a multiple of 8, K of 16.
    ``stable_weight``: the weight and its scales were written before the previous kernel on
    the stream began (``LINEAR_STABLE_WEIGHT``), so they may be fetched ahead of its end."""
    rows, k, stride = _check_rows("linear_fp8", x, FP8_DTYPE)
    if weight.ndim != 2 or weight.shape[1] != k:
        raise ValueError("linear_fp8 expects x [T, K] and weight [N, K]")
    n = weight.shape[0]
    index = x.get_device()
    blocks = -(-k // FP8_BLOCK)
    tall = -(-n // FP8_BLOCK)
    if not (weight.dtype is FP8_DTYPE and x_scale.dtype is weight_scale.dtype is torch.float32
            and x_scale.shape == (rows, blocks) and weight_scale.shape == (tall, blocks)
            and weight.get_device() == x_scale.get_device() == weight_scale.get_device() == index
            and weight.is_contiguous() and x_scale.is_contiguous() and weight_scale.is_contiguous()):
        _check_dense("linear_fp8", "weight", weight, (n, k), FP8_DTYPE, index)
        _check_dense("linear_fp8", "x_scale", x_scale, (rows, blocks), torch.float32, index)
        _check_dense("linear_fp8", "weight_scale", weight_scale, (tall, blocks), torch.float32, index)
    res_ptr, res_stride = None, 0
    if epilogue == _lib.EPI_ADD:
        if (residual is None or residual.shape != (rows, n) or residual.dtype is not torch.bfloat16
                or residual.get_device() != index or (residual.stride(1) != 1 and n > 1)):
            raise ValueError("the add epilogue needs a bf16 residual [rows, n] with contiguous rows")
        res_ptr, res_stride = residual.data_ptr(), residual.stride(0) if rows > 1 else n
    if out is None:
        out = _empty_rows(x, rows, n, torch.bfloat16)
        out_stride = n
    else:
        if (out.shape != (rows, n) or out.dtype is not torch.bfloat16 or out.get_device() != index
                or (out.stride(1) != 1 and n > 1)):
            raise ValueError("linear_fp8 output must be bf16 [rows, n] with contiguous rows")
        out_stride = out.stride(0) if rows > 1 else n
    if rows:
        _launch(index, "aiosb_linear_fp8", x.data_ptr(), stride, x_scale.data_ptr(), rows, k, weight.data_ptr(),
                weight_scale.data_ptr(), n, out.data_ptr(), out_stride,
                epilogue | _lib.LINEAR_STABLE_WEIGHT if stable_weight else epilogue, res_ptr, res_stride,
                _status_pointer(index))
    return out


def linear_fp8_plan(rows: int, n: int, k: int, sms: int = 0) -> tuple[int, int, int]:
    """How ``linear_fp8`` runs a size on a device of `sms` SMs (0: the current one): token
    rows and features of a tile, and the parts that k is split into."""
    plan = (ctypes.c_int32 * 3)()
    _lib.call("aiosb_linear_fp8_plan", rows, n, k, sms, ctypes.addressof(plan))
    return tuple(plan)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attention_decode(
    *,
    out: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    row_table: torch.Tensor,
    seq_lens: torch.Tensor,
    positions: torch.Tensor,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    scale: float,
    qkv: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
    q_norm_w: torch.Tensor | None = None,
    k_norm_w: torch.Tensor | None = None,
    eps: float = 1e-6,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    out_loc: torch.Tensor | None = None,
    prefix_len: torch.Tensor | None = None,
    active: torch.Tensor | None = None,
    stable_history: bool | int = False,
    staged_prefix: int = 0,
) -> torch.Tensor:
    """Decode attention. ``stable_history`` (fused ``qkv`` mode): the row table,
    prefix length, page-table entries before each row's current position and their
    K/V were written before the previous kernel on the stream began, so the kernel
    may stage them before waiting on that kernel. ``True`` / ``HISTORY_STAGED``:
    each row reads its keys itself; ``HISTORY_PREFIX_ONCE``: the rows of a KV head
    read the shared prefix once between them (a cluster of up to 8 rows).
    ``staged_prefix``: a bound on the prefix length (0: 128); the kernel stages that
    many prefix keys before its wait and sizes its shared memory by it."""
    rows = out.shape[0]
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    src = qkv if qkv is not None else q
    _lib.call(
        "aiosb_attention_decode",
        _ptr(qkv),
        qkv.stride(0) if qkv is not None else 0,
        _ptr(q),
        q.stride(0) if q is not None else 0,
        _ptr(q_norm_w),
        _ptr(k_norm_w),
        float(eps),
        _ptr(cos),
        _ptr(sin),
        cos.shape[0] if cos is not None else 0,
        positions.data_ptr(),
        _ptr(out_loc),
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        num_slots,
        page_table.data_ptr(),
        page_table.stride(0),
        row_table.data_ptr(),
        seq_lens.data_ptr(),
        _ptr(prefix_len),
        _ptr(active),
        int(stable_history),
        int(staged_prefix),
        rows,
        num_qo_heads,
        num_kv_heads,
        head_dim,
        float(scale),
        out.data_ptr(),
        out.stride(0),
        status_word(src.device).data_ptr(),
        _stream(src.device),
    )
    return out


def qk_norm_rope_store(
    *,
    qkv: torch.Tensor,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    q_norm_w: torch.Tensor,
    k_norm_w: torch.Tensor,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    out_loc: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    q_out: torch.Tensor,
) -> torch.Tensor:
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    _lib.call(
        "aiosb_qk_norm_rope_store",
        qkv.data_ptr(),
        qkv.stride(0),
        qkv.shape[0],
        num_qo_heads,
        num_kv_heads,
        head_dim,
        q_norm_w.data_ptr(),
        k_norm_w.data_ptr(),
        float(eps),
        cos.data_ptr(),
        sin.data_ptr(),
        cos.shape[0],
        positions.data_ptr(),
        out_loc.data_ptr(),
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        num_slots,
        q_out.data_ptr(),
        q_out.stride(0),
        status_word(qkv.device).data_ptr(),
        _stream(qkv.device),
    )
    return q_out


FUSED_PREFILL_MAX_TOKENS = 64  # new tokens per request on the fused prefill


def attention_prefill_fused(
    *,
    qkv: torch.Tensor,
    out: torch.Tensor,
    q_norm_w: torch.Tensor,
    k_norm_w: torch.Tensor,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    out_loc: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    meta: torch.Tensor,
    num_requests: int,
    num_tiles: int,
    tile_tokens: int,
    max_q_len: int,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    scale: float,
) -> torch.Tensor:
    """``qk_norm_rope_store`` and ``attention_prefill`` in one launch, for
    requests of at most FUSED_PREFILL_MAX_TOKENS new tokens whose cached keys were
    written by earlier launches; ``meta`` as for ``attention_prefill``. The output
    and the stored K/V equal the two-call path bit for bit."""
    _require_cuda(qkv, out, k_cache, v_cache, page_table, meta, what="attention_prefill_fused")
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    base = meta.data_ptr()
    r = num_requests * 4
    _lib.call(
        "aiosb_attention_prefill_fused",
        qkv.data_ptr(), qkv.stride(0), q_norm_w.data_ptr(), k_norm_w.data_ptr(), float(eps),
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(), out_loc.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), num_slots, page_table.data_ptr(), page_table.stride(0),
        base, base + r, base + 2 * r, base + 3 * r, base + 4 * r, base + 4 * r + num_tiles * 4,
        num_tiles, tile_tokens, max_q_len, num_qo_heads, num_kv_heads, head_dim, float(scale),
        out.data_ptr(), out.stride(0), status_word(qkv.device).data_ptr(), _stream(qkv.device),
    )
    return out


def prefill_tile_tokens(num_qo_heads: int, num_kv_heads: int) -> int:
    n = _lib.load().aiosb_prefill_tile_tokens(num_qo_heads, num_kv_heads)
    if n <= 0:
        raise ValueError("unsupported head grouping for prefill attention")
    return n


def attention_prefill(
    *,
    q: torch.Tensor,
    out: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    meta: torch.Tensor,
    num_requests: int,
    num_tiles: int,
    tile_tokens: int,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    scale: float,
) -> torch.Tensor:
    """``meta`` is one int32 device tensor holding, back to back, the request
    arrays q_start, q_len, cached_len, table_row ([num_requests] each) and the
    tile arrays tile_req, tile_q0 ([num_tiles] each)."""
    num_slots = k_cache.numel() // (num_kv_heads * head_dim)
    base = meta.data_ptr()
    r = num_requests * 4
    _lib.call(
        "aiosb_attention_prefill",
        q.data_ptr(),
        q.stride(0),
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        num_slots,
        page_table.data_ptr(),
        page_table.stride(0),
        base,
        base + r,
        base + 2 * r,
        base + 3 * r,
        base + 4 * r,
        base + 4 * r + num_tiles * 4,
        num_tiles,
        tile_tokens,
        num_qo_heads,
        num_kv_heads,
        head_dim,
        float(scale),
        out.data_ptr(),
        out.stride(0),
        status_word(q.device).data_ptr(),
        _stream(q.device),
    )
    return out


def prefill_meta(
    q_lens: list[int], cached_lens: list[int], table_rows: list[int], tile_tokens: int
) -> tuple[list[int], int]:
    """Host-side request/tile arrays for :func:`attention_prefill`."""
    q_start, acc = [], 0
    tile_req, tile_q0 = [], []
    for i, n in enumerate(q_lens):
        q_start.append(acc)
        acc += n
        for q0 in range(0, n, tile_tokens):
            tile_req.append(i)
            tile_q0.append(q0)
    return [*q_start, *q_lens, *cached_lens, *table_rows, *tile_req, *tile_q0], len(tile_req)


# ---------------------------------------------------------------------------
# Drafted token trees (speculative decoding)
# ---------------------------------------------------------------------------
TREE_MAX_NODES = 1024  # nodes of a tree


def _check_ints(what: str, name: str, t: torch.Tensor, size: int, index: int, dtype: torch.dtype = torch.int32) -> None:
    if t.dtype is not dtype or t.shape != (size,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} tensor of {size} on cuda:{index}")


def _check_trees(what: str, tree_start: torch.Tensor, index: int) -> int:
    """The number of trees."""
    if tree_start.ndim != 1 or tree_start.shape[0] < 1:
        raise ValueError(f"{what}: tree_start must have shape [requests + 1]")
    size = tree_start.shape[0]
    if tree_start.dtype is not torch.int32 or tree_start.get_device() != index or not tree_start.is_contiguous():
        raise ValueError(f"{what}: tree_start must be a contiguous int32 tensor on cuda:{index}")
    return size - 1


def draft_tree(
    parents: torch.Tensor,
    tree_start: torch.Tensor,
    *,
    max_nodes: int,
    cached_lens: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The ancestors' bits and the positions of drafted trees' nodes.

    Tree r is rows ``tree_start[r]`` to ``tree_start[r + 1]`` (int32, ascending); node 0 is the
    last token that is known, ``parents`` (int32) the number of each node's parent in its tree,
    less than its own, or -1. Returns ``mask`` (int32 [tokens, ceil(max_nodes / 32)]: bit j is set
    if node j is the node or an ancestor of it) and ``positions`` (int32: ``cached_lens[r]`` + the
    number of ancestors). ``max_nodes``: a bound on the nodes of a tree, at most 1024. Rows behind
    the last tree are left as they were."""
    if not parents.is_cuda:
        raise ValueError("draft_tree requires CUDA tensors")
    if parents.ndim != 1:
        raise ValueError("draft_tree: parents must have shape [tokens]")
    if not 1 <= max_nodes <= TREE_MAX_NODES:
        raise ValueError(f"draft_tree: max_nodes must be in [1, {TREE_MAX_NODES}]")
    tokens, index, words = parents.shape[0], parents.get_device(), (max_nodes + 31) // 32
    _check_ints("draft_tree", "parents", parents, tokens, index)
    requests = _check_trees("draft_tree", tree_start, index)
    if cached_lens is not None:
        _check_ints("draft_tree", "cached_lens", cached_lens, requests, index)
    if mask is None:
        mask = _empty_rows(parents, tokens, words, torch.int32)
    else:
        _check_dense("draft_tree", "mask", mask, (tokens, words), torch.int32, index)
    if positions is None:
        positions = _empty_vector(parents, tokens, torch.int32)
    else:
        _check_ints("draft_tree", "positions", positions, tokens, index)
    if tokens and requests:
        _launch(index, "aiosb_draft_tree", parents.data_ptr(), tokens, tree_start.data_ptr(), requests, words,
                _ptr(cached_lens), mask.data_ptr(), positions.data_ptr(), _status_pointer(index))
    return mask, positions


def attention_tree(
    *,
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    row_table: torch.Tensor,
    cached_lens: torch.Tensor,
    tree_start: torch.Tensor,
    tree_mask: torch.Tensor,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    scale: float,
    max_cached: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of drafted trees over the paged cache (``draft_tree`` for the arguments of the
    trees). q and out are bf16 [tokens, Hq * d], rows may be strided; the nodes' own K/V are in
    the cache (``qk_norm_rope_store``). Node i of request r sees the first ``cached_lens[r]``
    entries of page-table row ``row_table[r]``, and entry ``cached_lens[r] + j`` for every set bit
    j of ``tree_mask[i]`` (int32 [tokens, words]; any bits). A node that sees nothing gets 0.
    ``max_cached``: a bound on ``cached_lens`` from which the split over the GPU is chosen (0: the
    page table's width)."""
    width = num_qo_heads * head_dim
    tokens, cols, q_stride = _check_rows("attention_tree", q, torch.bfloat16)
    index = q.get_device()
    if cols != width:
        raise ValueError("attention_tree: q must have shape [tokens, num_qo_heads * head_dim]")
    if out is None:
        out, out_stride = _empty_rows(q, tokens, width, torch.bfloat16), width
    else:
        rows, cols, out_stride = _check_rows("attention_tree", out, torch.bfloat16)
        if rows != tokens or cols != width or out.get_device() != index:
            raise ValueError("attention_tree: out must match q")
    slots = k_cache.shape[0]
    cache = (slots, num_kv_heads, head_dim)
    requests = tree_start.shape[0] - 1 if tree_start.ndim == 1 else -1
    words = tree_mask.shape[1] if tree_mask.ndim == 2 else -1
    if not (k_cache.dtype is v_cache.dtype is torch.bfloat16 and k_cache.shape == cache and v_cache.shape == cache
            and k_cache.is_contiguous() and v_cache.is_contiguous() and requests >= 0 and words >= 0
            and tree_start.dtype is row_table.dtype is cached_lens.dtype is tree_mask.dtype is page_table.dtype
            is torch.int32 and row_table.shape == (requests,) and cached_lens.shape == (requests,)
            and tree_mask.shape == (tokens, words) and page_table.ndim == 2
            and (page_table.stride(1) == 1 or page_table.shape[1] <= 1) and tree_start.is_contiguous()
            and row_table.is_contiguous() and cached_lens.is_contiguous() and tree_mask.is_contiguous()
            and k_cache.get_device() == v_cache.get_device() == tree_start.get_device() == row_table.get_device()
            == cached_lens.get_device() == tree_mask.get_device() == page_table.get_device() == index):
        _refuse_attention_tree(index, tokens, cache, k_cache, v_cache, page_table, row_table, cached_lens, tree_start,
                               tree_mask)
    table_rows, table_width = page_table.shape
    if tokens and requests:
        work, size = None, 0
        # the library's rule for whole requests to a CTA, which take no work area
        if (max_cached or table_width) > 128 or tokens * num_qo_heads > 24000:
            with torch.cuda.device(index) if index != torch._C._cuda_getDevice() else nullcontext():
                size = _lib.load().aiosb_attention_tree_work_bytes(
                    tokens, requests, words, max_cached or table_width, num_qo_heads, num_kv_heads, head_dim)
            work = _empty_vector(q, size, torch.uint8) if size else None
        _launch(index, "aiosb_attention_tree", q.data_ptr(), q_stride, tokens, k_cache.data_ptr(), v_cache.data_ptr(),
                slots, page_table.data_ptr(), page_table.stride(0) if table_rows > 1 else table_width, table_rows,
                table_width, row_table.data_ptr(), cached_lens.data_ptr(), tree_start.data_ptr(), requests,
                tree_mask.data_ptr(), words, max_cached, num_qo_heads, num_kv_heads, head_dim, scale,
                out.data_ptr(), out_stride, _ptr(work), size, _status_pointer(index))
    return out


def _refuse_attention_tree(index, tokens, cache, k_cache, v_cache, page_table, row_table, cached_lens, tree_start,
                           tree_mask) -> None:
    """Names the argument that attention_tree does not take."""
    what = "attention_tree"
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dtype is not torch.bfloat16 or t.shape != cache or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous bf16 [slots, num_kv_heads, head_dim] tensor on "
                             f"cuda:{index}")
    requests = _check_trees(what, tree_start, index)
    _check_ints(what, "row_table", row_table, requests, index)
    _check_ints(what, "cached_lens", cached_lens, requests, index)
    if tree_mask.ndim != 2:
        raise ValueError(f"{what}: tree_mask must have shape [tokens, words]")
    _check_dense(what, "tree_mask", tree_mask, (tokens, tree_mask.shape[1]), torch.int32, index)
    raise ValueError(f"{what}: page_table must be an int32 tensor of contiguous rows on cuda:{index}")


def verify_draft(
    logits: torch.Tensor,
    draft_tokens: torch.Tensor,
    parents: torch.Tensor,
    tree_start: torch.Tensor,
    accept_uniforms: torch.Tensor | None = None,
    sample_uniforms: torch.Tensor | None = None,
    *,
    temperature: float = 1.0,
    greedy: bool = False,
    draft_probs: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted nodes stay, judged against the target model, and the token after them.

    ``logits`` (bf16 or fp32 [tokens, vocab]): row i is the target's distribution after node i;
    ``draft_tokens`` (int64): the nodes' tokens; the trees as for ``draft_tree``. From the root
    on, a node's children are tried in order: child c stays if ``accept_uniforms[c] * q(x) *
    sum(r) < r(x)``, where r is softmax(logits / temperature) less what the rejected ones took,
    and q is ``draft_probs`` (fp32 [tokens, vocab]; row i: the distribution that i's children were
    drawn from, independently) or 1 without it (distinct proposals). A rejection that would leave
    nothing (a certain token, a uniform of 1) leaves r as it was. With no child left the next
    token is drawn from r by inverse CDF with ``sample_uniforms``. What is kept has the target's
    distribution. ``greedy``: children and next token by argmax (the lowest id of equal ones).
    A sampler's filters (top-k, forbidden ids) go in as logits of -inf. Sampling takes up to 262144
    ids and temperatures in [1e-6, 1e6].

    Returns ``accepted`` (int32 [requests]: nodes behind the root that stay), ``next_token``
    (int64 [requests]; -1 where there is no tree, or a row of logits or probabilities that was read
    is no distribution) and ``order`` (int32
    [tokens]: each tree's node numbers, the path from the root first, then the others; undefined
    behind the last tree)."""
    if not logits.is_cuda:
        raise ValueError("verify_draft requires CUDA tensors")
    fp32 = logits.dtype is torch.float32
    if logits.ndim != 2 or not (fp32 or logits.dtype is torch.bfloat16):
        raise ValueError("verify_draft: logits must be a bf16 or fp32 tensor of shape [tokens, vocab]")
    tokens, vocab = logits.shape
    index = logits.get_device()
    stride, inner = logits.stride()
    if vocab > 1 and inner != 1:
        raise ValueError("verify_draft: logits rows must be contiguous")
    _check_ints("verify_draft", "draft_tokens", draft_tokens, tokens, index, torch.int64)
    _check_ints("verify_draft", "parents", parents, tokens, index)
    requests = _check_trees("verify_draft", tree_start, index)
    accept = sample = probs = None
    probs_stride = 0
    if not greedy:
        if accept_uniforms is None or sample_uniforms is None:
            raise ValueError("verify_draft: sampling needs accept_uniforms and sample_uniforms")
        _check_ints("verify_draft", "accept_uniforms", accept_uniforms, tokens, index, torch.float32)
        _check_ints("verify_draft", "sample_uniforms", sample_uniforms, requests, index, torch.float32)
        accept, sample = accept_uniforms.data_ptr(), sample_uniforms.data_ptr()
    if draft_probs is not None:
        if greedy:
            raise ValueError("verify_draft: greedy verification takes no draft_probs")
        if (draft_probs.dtype is not torch.float32 or draft_probs.shape != (tokens, vocab)
                or draft_probs.get_device() != index or (vocab > 1 and draft_probs.stride(1) != 1)):
            raise ValueError("verify_draft: draft_probs must be an fp32 [tokens, vocab] tensor with contiguous rows "
                             f"on cuda:{index}")
        probs, probs_stride = draft_probs.data_ptr(), draft_probs.stride(0) if tokens > 1 else vocab
    accepted = _empty_vector(logits, requests, torch.int32)
    next_token = _empty_vector(logits, requests, torch.int64)
    order = _empty_vector(logits, tokens, torch.int32)
    if requests:
        _launch(index, "aiosb_verify_draft", logits.data_ptr(), fp32, stride if tokens > 1 else vocab, tokens, vocab,
                draft_tokens.data_ptr(), parents.data_ptr(), tree_start.data_ptr(), requests, accept, sample,
                temperature, bool(greedy), probs, probs_stride, accepted.data_ptr(), next_token.data_ptr(),
                order.data_ptr(), _status_pointer(index))
    return accepted, next_token, order


# ---------------------------------------------------------------------------
# Sampler / uniforms / slot FIFO
# ---------------------------------------------------------------------------
def sample(
    logits: torch.Tensor,
    *,
    temperature: float,
    top_k: int,
    top_p: float,
    greedy: bool,
    uniforms: torch.Tensor | None,
    forbidden: torch.Tensor | None = None,
    forbidden_rows: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    rows, vocab = logits.shape
    dev = logits.device
    tok = torch.empty((rows, 1), dtype=torch.int64, device=dev)
    lp = torch.empty((rows, 1), dtype=torch.float32, device=dev)
    _lib.call(
        "aiosb_sample",
        logits.data_ptr(),
        rows,
        vocab,
        logits.stride(0),
        float(temperature),
        int(top_k),
        float(top_p),
        int(bool(greedy)),
        _ptr(uniforms),
        _ptr(forbidden),
        0 if forbidden is None else forbidden.numel(),
        _ptr(forbidden_rows),
        0 if forbidden_rows is None else forbidden_rows.shape[1],
        tok.data_ptr(),
        lp.data_ptr(),
        status_word(dev).data_ptr(),
        _stream(dev),
    )
    return tok, lp


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """log_softmax(logits.float())[r, targets[r]] per row, fp32."""
    rows, vocab = logits.shape
    t = targets.to(device=logits.device, dtype=torch.int64).contiguous()
    out = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _lib.call("aiosb_token_logprobs", logits.data_ptr(), rows, vocab, logits.stride(0), t.data_ptr(),
              out.data_ptr(), status_word(logits.device).data_ptr(), _stream(logits.device))
    return out


def stateless_uniforms_device(seeds: torch.Tensor, steps: int) -> torch.Tensor:
    out = torch.empty((seeds.numel(), steps), dtype=torch.float32, device=seeds.device)
    _lib.call("aiosb_stateless_uniforms", seeds.data_ptr(), seeds.numel(), steps, out.data_ptr(), _stream(seeds.device))
    return out


def slot_alloc(ring: torch.Tensor, head: int, n: int) -> torch.Tensor:
    out = torch.empty(n, dtype=torch.int32, device=ring.device)
    _lib.call("aiosb_slot_alloc", ring.data_ptr(), ring.numel(), head, n, out.data_ptr(), _stream(ring.device))
    return out


def slot_free(ring: torch.Tensor, tail: int, slots: torch.Tensor) -> None:
    slots = slots.to(torch.int32).contiguous()
    _lib.call("aiosb_slot_free", ring.data_ptr(), ring.numel(), tail, slots.data_ptr(), slots.numel(), _stream(ring.device))


def slot_free_range(ring: torch.Tensor, begin: int, n: int, tail: int) -> None:
    _lib.call("aiosb_slot_free_range", ring.data_ptr(), ring.numel(), begin, n, tail, _stream(ring.device))
