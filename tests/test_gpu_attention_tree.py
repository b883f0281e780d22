"""attention_tree against a plain restatement in fp64, within the roundings that the kernel makes."""

from __future__ import annotations

import pytest
import torch

from aios_b200.kernel import ops
from tests import draft_reference as ref

pytestmark = pytest.mark.gpu


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, sizes, cached, hq=4, hkv=2, d=64, kind="mixed", page=1, seed=0, spread=2.0, extra=0, words=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.sizes, self.cached_list, self.hq, self.hkv, self.d = sizes, cached, hq, hkv, d
        tokens = sum(sizes) + extra
        lens = [c + n for c, n in zip(cached, sizes)]
        pages = [-(-n // page) for n in lens]
        count = max(1, sum(pages))
        order = torch.randperm(count, generator=g, device="cuda")
        self.table = torch.full((len(sizes) + 2, max(lens, default=0) + 5), -3, dtype=torch.int32, device="cuda")
        self.row_list = torch.randperm(len(sizes) + 2, generator=g, device="cuda")[: len(sizes)].tolist()
        at = 0
        for row, n, p in zip(self.row_list, lens, pages):
            slots = (order[at : at + p, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n]
            self.table[row, :n] = slots.to(torch.int32)
            at += p
        self.k = torch.randn((count * page, hkv, d), generator=g, device="cuda").to(torch.bfloat16)
        self.v = torch.randn((count * page, hkv, d), generator=g, device="cuda").to(torch.bfloat16)
        self.q = (spread * torch.randn((tokens, hq * d), generator=g, device="cuda")).to(torch.bfloat16)
        self.rows, self.cached = _i32(self.row_list), _i32(cached)
        self.start = _i32(ref.starts(sizes))
        words = words or (max(sizes, default=1) + 31) // 32 or 1
        mask, _ = ref.tree_bits(ref.trees(sizes, kind, seed), words)
        self.mask = torch.full((tokens, words), -1, dtype=torch.int32, device="cuda")
        self.mask[: sum(sizes)] = mask.cuda()
        self.scale = d**-0.5

    def run(self, **kw):
        args = dict(q=self.q, k_cache=self.k, v_cache=self.v, page_table=self.table, row_table=self.rows,
                    cached_lens=self.cached, tree_start=self.start, tree_mask=self.mask, num_qo_heads=self.hq,
                    num_kv_heads=self.hkv, head_dim=self.d, scale=self.scale)
        args.update(kw)
        return ops.attention_tree(**args)

    def check_every_way(self):
        """Whole requests to a CTA, and keys dealt over the SMs (the bound on the histories chooses)."""
        for bound in (1, 1 << 20):
            self.check(self.run(max_cached=bound))

    def check(self, got):
        n = sum(self.sizes)
        want, mag, top = ref.attention(self.q[:n], self.k, self.v, self.table, self.row_list, self.cached_list, self.sizes,
                                       self.mask[:n], self.hq, self.hkv, self.d, self.scale)
        keys = max([c + n for c, n in zip(self.cached_list, self.sizes)], default=0)
        tol = ref.attention_tolerance(want, mag, top, keys, self.d)
        err = (got[:n].double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
        ops.check_status(torch.device("cuda", 0))


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (12, 4), (8, 1), (7, 7), (64, 1)])
@pytest.mark.parametrize("page", [1, 16])
def test_heads(cuda_device, d, heads, page) -> None:
    c = Case([5, 1, 13], [37, 0, 130], *heads, d, page=page, seed=d)
    c.check_every_way()


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 128, 200])
@pytest.mark.parametrize("cached", [0, 1, 63, 64, 65, 127, 128, 300])
def test_sizes(cuda_device, nodes, cached) -> None:
    c = Case([nodes], [cached], 6, 2, 64, seed=nodes)
    c.check_every_way()


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("kind", ["chain", "star", "mixed"])
def test_ragged_batches(cuda_device, d, kind) -> None:
    sizes = [3, 0, 64, 1, 40, 7, 0, 17, 100]
    cached = [500, 20, 0, 1, 1000, 3, 0, 129, 64]
    c = Case(sizes, cached, 8, 2, d, kind=kind, page=16, seed=7)
    c.check_every_way()


@pytest.mark.parametrize("d,heads,requests,nodes,cached", [
    (128, (32, 8), 1, 64, 20000), (128, (8, 8), 2, 1, 9001), (64, (12, 4), 3, 9, 7777), (96, (8, 2), 2, 150, 5000),
    (64, (64, 1), 1, 33, 12345), (128, (4, 1), 40, 4, 3500),
])
def test_long_histories(cuda_device, d, heads, requests, nodes, cached) -> None:
    sizes = [max(1, nodes - 3 * i % nodes) for i in range(requests)]
    lens = [cached if i == 0 else cached * (i % 7) // 9 for i in range(requests)]
    c = Case(sizes, lens, *heads, d, page=16, seed=cached)
    c.check(c.run())
    c.check(c.run(max_cached=cached))


def test_the_largest_tree(cuda_device) -> None:
    c = Case([1024, 1000], [70, 2000], 4, 2, 64, seed=2)
    c.check_every_way()


def test_any_bits(cuda_device) -> None:
    """Bits that are no tree's, beyond the tree's size, and nodes that see nothing."""
    g = torch.Generator().manual_seed(3)
    c = Case([40, 20, 9], [0, 100, 0], 4, 2, 64, seed=5)
    n = sum(c.sizes)
    bits = torch.randint(-(1 << 31), 1 << 31, (n, 2), generator=g)
    bits[5] = 0
    bits[40] = 0  # its history alone
    bits[62] = 0
    bits[10, 0], bits[10, 1] = 0, 1 << 30  # past the tree's 40 nodes: nothing
    c.mask[:n] = bits.to(torch.int32).cuda()
    for bound in (1, 1 << 20):
        out = torch.full_like(c.q, 7.0)
        c.run(out=out, max_cached=bound)
        c.check(out)
        assert (out[5] == 0).all() and (out[62] == 0).all() and (out[10] == 0).all() and (out[40] != 0).any()


def test_rows_behind_the_last_tree_and_strides(cuda_device) -> None:
    c = Case([5, 9], [40, 3], 4, 2, 64, seed=1, extra=6)
    q = torch.full((20, 4 * 64 + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[:, 8:264] = c.q
    out = torch.full((20, 4 * 64 + 40), 3.0, dtype=torch.bfloat16, device="cuda")
    table = torch.full((4, c.table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    table[:, : c.table.shape[1]] = c.table
    for bound in (1, 1 << 20):
        out.fill_(3)
        c.run(q=q[:, 8:264], out=out[:, 16:272], page_table=table[:, : c.table.shape[1]], max_cached=bound)
        c.check(out[:, 16:272])
        assert (out[14:] == 3).all() and (out[:, :16] == 3).all() and (out[:, 272:] == 3).all()


@pytest.mark.parametrize("nodes", [5, 20, 100])
def test_a_query_that_is_no_number_stays_in_its_row(cuda_device, nodes) -> None:
    c = Case([nodes, nodes], [900, 40], 4, 2, 64, seed=6)
    for bound in (1, 1 << 20):
        clean = c.run(max_cached=bound)
        kept = c.q[3, 64].clone()
        c.q[3, 64] = float("nan")  # head 1 of node 3
        got = c.run(max_cached=bound)
        c.q[3, 64] = kept
        assert torch.isnan(got[3, 64:128]).all()
        got[3, 64:128] = clean[3, 64:128]
        assert torch.equal(got, clean)


def test_more_requests_than_a_warp_has_lanes(cuda_device) -> None:
    """Ranges that start among hundreds of requests of unlike sizes, some of them empty."""
    sizes = [(7 * i) % 11 for i in range(300)]
    cached = [(131 * i) % 700 if i % 5 else 0 for i in range(300)]
    c = Case(sizes, cached, 4, 2, 64, seed=8)
    c.check_every_way()


def test_many_rows_over_short_histories(cuda_device) -> None:
    """Enough rows for the tensor cores, whatever the bound on the histories says."""
    c = Case([60] * 64, [(5 * i) % 40 for i in range(64)], 8, 2, 64, seed=8)
    c.check_every_way()


def test_every_kind_of_unit_in_one_batch(cuda_device) -> None:
    """Units of up to 16, 32, 128 and 256 rows, and of 256 with a rest of each kind, cut at any place."""
    sizes = [3, 8, 30, 60, 64 + 3, 64 + 30, 128 + 50]
    for cached in ([3000] * 7, [100, 5000, 1, 700, 2000, 0, 333]):
        c = Case(sizes, cached, 8, 2, 128, seed=9, page=16)
        c.check_every_way()


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("cached", [0, 30, 700])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("bound", [1, 1 << 20])
def test_what_a_node_does_not_see_does_not_reach_it(cuda_device, d, cached, value, bound) -> None:
    sizes = [20, 50]
    c = Case(sizes, [cached, cached], 4, 2, d, kind="star", seed=11)
    clean = c.run(max_cached=bound)
    # node 7 of the first tree, nodes 3 and 45 of the second: only they see themselves
    hit = [(0, 7), (1, 3), (1, 45)]
    for r, j in hit:
        slot = int(c.table[c.row_list[r], cached + j])
        c.v[slot, :, 5] = value
        c.k[slot, 0, 2] = value
    got = c.run(max_cached=bound)
    touched = [r * 20 + j for r, j in hit]
    rest = [i for i in range(70) if i not in touched]
    assert torch.equal(got[rest], clean[rest])
    # head group 1: its keys are finite, so that only the value's own column is not
    for i in touched:
        x = got[i].view(4, d)[2:]
        assert not torch.isfinite(x[:, 5]).any()
        assert torch.isfinite(x[:, :5]).all() and torch.isfinite(x[:, 6:]).all()
        if value == value:
            assert (x[:, 5] == value).all()
    ops.check_status(cuda_device)


def test_unused_pool_slots_and_table_entries_do_not_matter(cuda_device) -> None:
    c = Case([6, 3], [50, 20], 4, 2, 64, page=16, seed=4)
    clean = c.run()
    used = torch.zeros(c.k.shape[0], dtype=torch.bool, device="cuda")
    for row, n, length in zip(c.row_list, c.sizes, c.cached_list):
        used[c.table[row, : length + n].long()] = True
    dealt = c.run(max_cached=1 << 20)
    c.k[~used] = float("nan")
    c.v[~used] = float("nan")
    assert torch.equal(c.run(), clean) and torch.equal(c.run(max_cached=1 << 20), dealt)


def test_a_large_score_and_equal_scores(cuda_device) -> None:
    c = Case([3], [200], 2, 1, 64, seed=9, spread=30.0)
    c.check_every_way()
    c.q.zero_()  # every key alike: a plain mean
    c.check_every_way()


def test_a_history_that_grows_in_score(cuda_device) -> None:
    """Every chunk of keys has larger scores than the one before: the rows' references move each time."""
    c = Case([9], [1500], 4, 2, 128, seed=2)
    order = c.table[c.row_list[0], :1500].long()
    c.q.copy_(c.q.abs() + 1)
    c.k[order] = (torch.arange(1500, device="cuda")[:, None, None] / 60).expand(1500, 2, 128).to(torch.bfloat16)
    c.check_every_way()
    c.k[order] = c.k[order.flip(0)]
    c.check_every_way()


def test_one_history_of_several_requests(cuda_device) -> None:
    """Two trees over the same page-table row, the same slots twice."""
    c = Case([4, 4], [100, 100], 4, 2, 64, seed=10)
    c.row_list = [c.row_list[0]] * 2
    c.rows = _i32(c.row_list)
    c.check(c.run())


@pytest.mark.parametrize("bound", [1, 1 << 20])
@pytest.mark.parametrize("what", ["slot", "row", "cached", "start", "width", "words"])
def test_numbers_outside_their_arrays_are_reported(cuda_device, what, bound) -> None:
    c = Case([4, 40], [100, 30], 4, 2, 64, seed=12)
    if what == "slot":
        c.table[c.row_list[0], 50] = c.k.shape[0]
    elif what == "row":
        c.rows[1] = 4
    elif what == "cached":
        c.cached[0] = -1
    elif what == "start":
        c.start[2] = 45
    elif what == "width":
        c.cached[1] = 1 << 30
    else:
        c.mask = c.mask[:, :1].contiguous()
    out = c.run(max_cached=bound)
    torch.cuda.synchronize()
    assert out.shape == c.q.shape
    with pytest.raises(RuntimeError, match="slot" if what == "slot" else "tree"):
        ops.check_status(cuda_device)


def test_refusals(cuda_device) -> None:
    c = Case([4, 4], [10, 3], 4, 2, 64)
    wide = torch.zeros(8, 512, dtype=torch.bfloat16, device="cuda")
    bad = [dict(q=c.q.float()), dict(q=c.q[:, :128]), dict(q=wide[:, ::2]), dict(out=c.q[:3]), dict(out=c.q.float()),
           dict(k_cache=c.k.float()), dict(v_cache=c.v[:5]), dict(k_cache=c.k[:, :1]), dict(row_table=c.rows.long()),
           dict(row_table=c.rows[:1]), dict(cached_lens=c.cached.cpu()), dict(tree_start=c.start.long()),
           dict(page_table=c.table.long()), dict(page_table=c.table.t()), dict(tree_mask=c.mask[:3]),
           dict(tree_mask=c.mask.long()), dict(tree_mask=c.mask[0]), dict(head_dim=32, num_qo_heads=8),
           dict(num_kv_heads=3), dict(q=torch.zeros(8, 260, dtype=torch.bfloat16, device="cuda")[:, 4:])]
    for change in bad:
        with pytest.raises(ValueError):
            c.run(**change)
    assert c.run(q=c.q[:0], tree_mask=c.mask[:0]).shape == (0, 256)


def test_same_bits_every_time_and_two_streams_at_once(cuda_device) -> None:
    cases = [Case([30, 7], [9000, 300], 8, 2, 128, seed=s) for s in (1, 2)]
    want = [c.run() for c in cases]
    for c, w in zip(cases, want):
        c.check(w)
        for _ in range(3):
            assert torch.equal(c.run(), w)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(c.run())
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_two_captured_graphs(cuda_device) -> None:
    """Graphs of different sizes, captured one after the other and replayed at the same time, with lengths
    that change between replays."""
    cases = [Case([30, 7], [9000, 300], 8, 2, 128, seed=1), Case([4], [20000], 8, 2, 128, seed=2)]
    side, graphs, outs = torch.cuda.Stream(), [], []
    for c in cases:
        c.run()
    torch.cuda.synchronize()
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(c.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cases]
    for lens in ([9000, 300, 20000], [77, 8000, 64]):
        cases[0].cached.copy_(_i32(lens[:2]))
        cases[1].cached.copy_(_i32(lens[2:]))
        cases[0].cached_list, cases[1].cached_list = lens[:2], lens[2:]
        for c in cases:  # every row long enough for either length
            for row in c.row_list:
                c.table[row] = torch.randint(0, c.k.shape[0], c.table[row].shape, device="cuda").to(torch.int32)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            c.check(o)


def test_on_another_stream_after_a_pending_write(cuda_device) -> None:
    c = Case([9], [3000], 8, 2, 64, seed=3)
    want = c.run()
    side = torch.cuda.Stream()
    q, c.q = c.q, torch.zeros_like(c.q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        c.q.copy_(q)
        got = c.run()
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_past_two_to_the_31(cuda_device) -> None:
    """A pool of more than 2^31 values: slots at its end."""
    slots = (1 << 31) // (8 * 128) + 4096
    k = torch.zeros(slots, 8, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    c = Case([5], [60], 8, 8, 128, seed=3)
    n = c.k.shape[0]
    k[-n:], v[-n:] = c.k, c.v
    shifted = torch.where(c.table >= 0, c.table + (slots - n), c.table)
    want = c.run()
    got = c.run(k_cache=k, v_cache=v, page_table=shifted)
    assert torch.equal(got, want)
