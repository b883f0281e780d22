"""Argument checks of the drafted trees' entry points: they run before any CUDA call, so every
refusal is seen on a CPU machine."""

from __future__ import annotations

import pytest
import torch

from aios_b200 import _lib
from aios_b200.kernel import ops

P = 1 << 20  # an aligned address that is never read: every call below is refused first
INV, UNS, MIS = _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_MISALIGNED


def _refused(name: str, good: dict, code: int, text: str, **changes) -> None:
    rc = getattr(_lib.load(), name)(*{**good, **changes}.values())
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


def test_draft_tree_refuses() -> None:
    name = "aiosb_draft_tree"
    good = dict(parents=P, tokens=4, start=P, requests=1, words=1, cached=None, mask=P, pos=P, status=None, stream=None)
    _refused(name, good, INV, "bad sizes", tokens=-1)
    _refused(name, good, INV, "bad sizes", requests=-1)
    _refused(name, good, INV, "bad sizes", tokens=1 << 31)
    _refused(name, good, UNS, "at most 1024", words=0)
    _refused(name, good, UNS, "at most 1024", words=33)
    for field in ("parents", "start", "mask", "pos"):
        _refused(name, good, INV, "null", **{field: None})
    fn = _lib.load().aiosb_draft_tree
    assert fn(*{**good, "tokens": 0, "parents": None}.values()) == _lib.OK
    assert fn(*{**good, "requests": 0, "start": None}.values()) == _lib.OK


ATTENTION = dict(q=P, qs=768, tokens=4, k=P, v=P, slots=64, table=P, ts=512, rows=4, width=512, row_table=P, cached=P,
                 start=P, requests=1, mask=P, words=1, max_cached=0, hq=12, hkv=4, d=64, scale=0.125, out=P, os=768,
                 work=P, work_bytes=1 << 40, status=None, stream=None)


def test_attention_tree_refuses() -> None:
    def call(code, text, **changes):
        _refused("aiosb_attention_tree", ATTENTION, code, text, **changes)

    call(INV, "divisible", hq=13)
    call(INV, "divisible", hkv=0)
    call(UNS, "head_dim", d=80)
    call(INV, "bad sizes", tokens=-1)
    call(INV, "bad sizes", max_cached=-1)
    for scale in (0.0, -0.125, float("inf"), float("nan")):
        call(INV, "bad sizes", scale=scale)
    call(UNS, "at most 1024", words=33)
    call(UNS, "at most 1024", words=0)
    call(UNS, "too many", hq=65 * 4, qs=65 * 256, os=65 * 256)
    call(UNS, "too many", requests=65536)
    call(UNS, "too many", width=(1 << 30) + 1, ts=1 << 31)
    call(INV, "row strides", qs=760)
    call(INV, "row strides", qs=772)
    call(INV, "row strides", os=760)
    call(INV, "row strides", os=769)
    call(INV, "page-table stride", ts=511)
    call(INV, "empty cache", slots=0)
    call(INV, "empty cache", rows=0)
    for field in ("q", "k", "v", "table", "row_table", "cached", "start", "mask", "out"):
        call(INV, "null", **{field: None})
    for field in ("q", "k", "v", "out"):
        call(MIS, "aligned", **{field: P + 8})
    fn = _lib.load().aiosb_attention_tree
    assert fn(*{**ATTENTION, "tokens": 0, "q": None}.values()) == _lib.OK
    assert fn(*{**ATTENTION, "requests": 0, "start": None}.values()) == _lib.OK


def test_verify_draft_refuses() -> None:
    name = "aiosb_verify_draft"
    good = dict(logits=P, fp32=0, ls=100, tokens=4, vocab=100, drafts=P, parents=P, start=P, requests=1, au=P, su=P,
                temperature=1.0, greedy=0, probs=None, ps=0, accepted=P, token=P, order=P, status=None, stream=None)
    _refused(name, good, INV, "bad sizes", tokens=-1)
    _refused(name, good, INV, "bad sizes", vocab=0)
    _refused(name, good, INV, "bad sizes", requests=1 << 29)
    _refused(name, good, UNS, "too large", vocab=262145, ls=262152)
    _refused(name, good, UNS, "too large", vocab=262138, ls=262138)  # rows anywhere on 16 bytes
    _refused(name, good, UNS, "too large", vocab=262144, ls=262144, logits=P + 2)
    _refused(name, good, UNS, "too large", vocab=1 << 31, ls=1 << 31, greedy=1)
    _refused(name, good, INV, "logits row stride", ls=99)
    _refused(name, good, INV, "temperature", temperature=0.0)
    _refused(name, good, INV, "temperature", temperature=-1.0)
    _refused(name, good, INV, "temperature", temperature=float("nan"))
    _refused(name, good, INV, "temperature", temperature=float("inf"))
    _refused(name, good, INV, "temperature", temperature=0.9e-6)
    _refused(name, good, INV, "temperature", temperature=1.1e6)
    _refused(name, good, INV, "greedy", greedy=1, probs=P, ps=100)
    _refused(name, good, INV, "draft_probs row stride", probs=P, ps=99)
    _refused(name, good, INV, "uniforms", au=None)
    _refused(name, good, INV, "uniforms", su=None)
    for field in ("logits", "drafts", "parents", "start", "accepted", "token", "order"):
        _refused(name, good, INV, "null", **{field: None})
    assert _lib.load().aiosb_verify_draft(*{**good, "requests": 0, "start": None}.values()) == _lib.OK


def test_wrappers_want_cuda_tensors() -> None:
    i, f = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.draft_tree(i, i, max_nodes=2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_tree(q=f, k_cache=f, v_cache=f, page_table=f, row_table=i, cached_lens=i, tree_start=i,
                           tree_mask=f, num_qo_heads=1, num_kv_heads=1, head_dim=8, scale=1.0)
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_draft(f, i.long(), i, i, greedy=True)


@pytest.mark.parametrize("bound", [1, 127, 128, 129, 5000])
@pytest.mark.parametrize("tokens", [1, 100, 3000, 3001])
def test_the_work_areas_rule_is_the_wrappers(bound: int, tokens: int) -> None:
    """attention_tree asks the library for a work area's size only where it needs one."""
    size = _lib.load().aiosb_attention_tree_work_bytes(tokens, 1, 1, bound, 8, 2, 64)
    assert (size > 0) == (bound > 128 or tokens * 8 > 24000)


@pytest.mark.parametrize("tokens", [1, 3000, 3001])
@pytest.mark.parametrize("width", [64, 128, 129, 4096])
def test_without_a_bound_the_work_area_is_enough_for_any_width(tokens: int, width: int) -> None:
    """max_cached 0 stands for the page table's width, which the query does not have: it names what the widest needs."""
    lib = _lib.load()
    size = lib.aiosb_attention_tree_work_bytes(tokens, 1, 1, 0, 12, 4, 64)
    assert size >= lib.aiosb_attention_tree_work_bytes(tokens, 1, 1, width, 12, 4, 64) and size > 0
    good = {**ATTENTION, "tokens": tokens, "width": width, "ts": width}
    if width > 128 or tokens * 12 > 24000:
        _refused("aiosb_attention_tree", good, INV, "work area", work_bytes=size - 1)
        _refused("aiosb_attention_tree", good, INV, "work area", work=P + 8, work_bytes=size)
