"""The operators of drafted token trees as they are measured: cases, inputs, plain forms and definitions.

A drafting model proposes a tree of tokens after each request's last token; the target
model runs over all nodes at once and keeps one path:

* ``draft_tree``: from each node's parent, the bits of its ancestors (and itself) and its position;
* ``attention_tree``: attention of the nodes over the request's paged cache and their ancestors;
* ``verify_draft``: which nodes stay, judged against the target's probabilities with given uniforms,
  and the token after them.

A tree's nodes follow one another (rows tree_start[r] .. tree_start[r + 1]); node 0 is the root, the
last token that is known; a parent comes before its children.
"""

from __future__ import annotations

import math
import random

import torch

own = False


def listed():
    return [
        # a keystroke's 8 drafted nodes over its prefix, S10 heads: latency
        {"name": "attention_keystroke", "op": "attention", "requests": 1, "nodes": 8, "cached": 32, "hq": 12, "hkv": 4,
         "d": 64, "page": 16, "ragged": False, "shape": 1},
        # a serving batch with short histories, ragged, S06 heads
        {"name": "attention_batch", "op": "attention", "requests": 16, "nodes": 26, "cached": 1900, "hq": 8, "hkv": 2,
         "d": 96, "page": 1, "ragged": True, "shape": 2},
        # one request with a very long history: the work has to be split along it
        {"name": "attention_long", "op": "attention", "requests": 1, "nodes": 64, "cached": 131071, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "ragged": False, "shape": 3},
        # short chains at many requests: bound by the cache's bytes
        {"name": "attention_chain", "op": "attention", "requests": 64, "nodes": 5, "cached": 8192, "hq": 12, "hkv": 4,
         "d": 64, "page": 1, "ragged": False, "shape": 4},
        # histories from tens to tens of thousands of tokens in one batch
        {"name": "attention_ragged", "op": "attention", "requests": 41, "nodes": 33, "cached": 40000, "hq": 16, "hkv": 2,
         "d": 128, "page": 16, "ragged": True, "shape": 5},
        # a large batch of wide trees: bytes and products weigh the same
        {"name": "attention_wide", "op": "attention", "requests": 32, "nodes": 64, "cached": 16384, "hq": 32, "hkv": 8,
         "d": 128, "page": 16, "ragged": False, "shape": 6},
        # a drafted chain of one request, S10 vocabulary: latency
        {"name": "verify_keystroke", "op": "verify", "requests": 1, "nodes": 5, "vocab": 16384, "chain": True,
         "probs": True, "greedy": False, "dtype": "bf16", "shape": 7},
        # greedy serving, odd vocabulary, fp32 logits
        {"name": "verify_greedy", "op": "verify", "requests": 24, "nodes": 13, "vocab": 50021, "chain": False,
         "probs": False, "greedy": True, "dtype": "fp32", "shape": 8},
        # trees of distinct proposals without the drafting model's probabilities
        {"name": "verify_tree", "op": "verify", "requests": 16, "nodes": 26, "vocab": 32001, "chain": False,
         "probs": False, "greedy": False, "dtype": "bf16", "shape": 9},
        # a large batch, a large vocabulary, trees drawn from the drafting model's probabilities
        {"name": "verify_large", "op": "verify", "requests": 64, "nodes": 24, "vocab": 131072, "chain": False,
         "probs": True, "greedy": False, "dtype": "bf16", "shape": 10},
        # one small tree before a forward: latency
        {"name": "tree_keystroke", "op": "tree", "requests": 1, "nodes": 8, "chain": False, "shape": 11},
        # a large batch of wide trees
        {"name": "tree_large", "op": "tree", "requests": 256, "nodes": 256, "chain": False, "shape": 12},
    ]


def _log(rng, low, high):
    """A whole number in [low, high], spread over the logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "verify", "verify", "tree"])
    shape = rng.randrange(1 << 30)
    while True:
        if op == "attention":
            hq, hkv = rng.choice([(12, 4), (8, 2), (32, 8), (16, 2), (8, 8), (16, 16), (28, 4)])
            c = {"op": op, "requests": _log(rng, 1, 64), "nodes": _log(rng, 1, 128), "cached": _log(rng, 1, 131072),
                 "hq": hq, "hkv": hkv, "d": rng.choice([64, 96, 128]), "page": rng.choice([1, 16]),
                 "ragged": rng.random() < 0.5, "shape": shape}
            keys = c["requests"] * (c["cached"] + c["nodes"])
            if keys * hkv * c["d"] <= 32 * 16448 * 8 * 128 and keys * c["nodes"] * hq * c["d"] <= 32 * 16448 * 64 * 32 * 128:
                return c
        elif op == "verify":
            c = {"op": op, "requests": _log(rng, 1, 64), "nodes": _log(rng, 1, 64), "vocab": _log(rng, 1000, 160000),
                 "chain": rng.random() < 0.3, "probs": rng.random() < 0.5, "greedy": rng.random() < 0.25,
                 "dtype": rng.choice(["bf16", "bf16", "fp32"]), "shape": shape}
            c["probs"] = c["probs"] and not c["greedy"]
            if c["requests"] * c["nodes"] * c["vocab"] <= 64 * 24 * 131072:
                return c
        else:
            return {"op": op, "requests": _log(rng, 1, 256), "nodes": _log(rng, 1, 256), "chain": rng.random() < 0.3,
                    "shape": shape}


TEMPERATURE = 0.8


def _trees(case, seed=0):
    """Sizes and parents of the case's trees: a chain, or every node hung below one of the 8 before it. The seed
    changes the parents."""
    rng = random.Random(case["shape"])
    most = case["nodes"]
    sizes = [most if i == 0 or not case.get("ragged", True) else rng.randint(max(1, most // 4), most)
             for i in range(case["requests"])]
    chain = case.get("chain", False)
    rng = random.Random(case["shape"] + 7 * seed)
    parents = []
    for n in sizes:
        parents += [-1 if i == 0 else i - 1 if chain else rng.randint(max(0, i - 8), i - 1) for i in range(n)]
    return sizes, parents


def _cached(case):
    rng = random.Random(case["shape"] + 1)
    if not case["ragged"]:
        return [case["cached"]] * case["requests"]
    return [case["cached"] if i == 0 else _log(rng, 1, case["cached"]) for i in range(case["requests"])]


def work(case):
    sizes, _ = _trees(case)
    tokens = sum(sizes)
    words = -(-case["nodes"] // 32)
    if case["op"] == "tree":
        return {"bytes": tokens * (4 + 4 * words + 4), "flops": tokens}
    if case["op"] == "attention":
        cached = _cached(case)
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        keys = sum(cached) + tokens
        moved = keys * (4 * hkv * d + 4) + tokens * (4 * hq * d + 4 * words)
        # every node sees its whole history and itself at least
        return {"bytes": moved, "flops": sum(4 * hq * d * n * (length + 1) for n, length in zip(sizes, cached))}
    # one row of logits a request at least, and the row that its drafts came from
    size = 2 if case["dtype"] == "bf16" else 4
    rows = case["requests"] * case["vocab"]
    return {"bytes": rows * (size + (4 if case["probs"] else 0)) + 20 * tokens, "flops": rows * 4}


def _extent(sizes, parents):
    """The trees' largest depth, and the most children of a node."""
    at, deepest, broadest = 0, 0, 0
    for n in sizes:
        depth, count = [0] * n, [0] * n
        for i in range(1, n):
            p = parents[at + i]
            depth[i] = depth[p] + 1
            count[p] += 1
        deepest, broadest = max(deepest, max(depth)), max(broadest, max(count))
        at += n
    return deepest, broadest


# ---- inputs ------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _starts(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    sizes, parents = _trees(case, seed if case["op"] == "tree" else 0)
    starts = _starts(sizes)
    deepest, broadest = _extent(sizes, parents)  # as the program that drafted the trees knows them
    state = {"case": case, "sizes": sizes, "parents": _ints(parents), "tree_start": _ints(starts), "deepest": deepest,
             "broadest": broadest}
    if case["op"] == "tree":
        state["cached"] = _ints([rng.randrange(40000) for _ in sizes])
        return state
    if case["op"] == "attention":
        return _prepare_attention(case, state, gen)
    return _prepare_verify(case, state, parents, starts, gen)


def _prepare_attention(case, state, gen):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    sizes, cached = state["sizes"], _cached(case)
    lens = [length + n for length, n in zip(cached, sizes)]
    tokens = sum(sizes)
    # the pool's pages in the order in which a busy server hands them out
    pages = [-(-n // page) for n in lens]
    count = sum(pages) + 3
    order = torch.randperm(count, generator=gen, device="cuda")
    table = torch.zeros((len(lens), max(lens) + 7), dtype=torch.int32, device="cuda")
    rows = torch.randperm(len(lens), generator=gen, device="cuda")
    at = 0
    row_list = rows.tolist()
    for row, n, p in zip(row_list, lens, pages):
        slots = (order[at : at + p, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:n]
        table[row, :n] = slots.to(torch.int32)
        at += p

    def keys():
        x = torch.randn((count * page, hkv, d), generator=gen, device="cuda", dtype=torch.bfloat16)
        x *= torch.exp(0.4 * torch.randn((1, hkv, d), generator=gen, device="cuda")).to(torch.bfloat16)
        return x

    state.update(
        k=keys(), v=keys(), table=table, rows=rows.to(torch.int32), cached=_ints(cached), cached_list=cached,
        row_list=row_list, scale=d**-0.5, max_cached=max(cached),
        # sharper than chance, as trained heads are
        q=(2 * torch.randn((tokens, hq * d), generator=gen, device="cuda")).to(torch.bfloat16),
        out=torch.empty((tokens, hq * d), dtype=torch.bfloat16, device="cuda"),
    )
    # the ancestors' bits, made once a forward and read by every layer
    state["mask"] = _plain_tree(state)["mask"]
    return state


def _prepare_verify(case, state, parents, starts, gen):
    vocab, tokens = case["vocab"], starts[-1]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = torch.empty((tokens, vocab), dtype=dtype, device="cuda")
    probs = torch.empty((tokens, vocab), device="cuda") if case["probs"] else None
    children = [[] for _ in range(tokens)]
    for r, n in enumerate(state["sizes"]):
        for i in range(1, n):
            children[starts[r] + parents[starts[r] + i]].append(starts[r] + i)
    most = max(1, max(len(c) for c in children))
    picks = torch.empty((tokens, most), dtype=torch.int64, device="cuda")
    for a in range(0, tokens, 128):  # the target's logits, and a drafting model that is near them
        b = min(tokens, a + 128)
        x = 2.5 * torch.randn((b - a, vocab), generator=gen, device="cuda")
        x += 6 * (torch.rand((b - a, vocab), generator=gen, device="cuda") < 8 / vocab)
        logits[a:b] = x.to(dtype)
        y = x + 0.6 * torch.randn((b - a, vocab), generator=gen, device="cuda")
        if probs is not None:  # children are drawn from the drafting model's distribution
            probs[a:b] = torch.softmax(y / TEMPERATURE, dim=1)
            picks[a:b] = torch.multinomial(probs[a:b], most, replacement=True, generator=gen)
        else:  # children are its likeliest tokens
            picks[a:b] = torch.topk(y, most, dim=1).indices
    where = [0] * tokens
    for row, nodes in enumerate(children):
        for rank, node in enumerate(nodes):
            where[node] = row * most + rank
    state.update(
        logits=logits, probs=probs, tokens=picks.view(-1)[torch.tensor(where).cuda()],
        accept=torch.rand(tokens, generator=gen, device="cuda"),
        sample=torch.rand(len(state["sizes"]), generator=gen, device="cuda"),
    )
    return state


# ---- plain forms -------------------------------------------------------------
def _owner(state):
    """The tree of each node, and the node's number in it."""
    tokens = state["parents"].numel()
    node = torch.arange(tokens, device="cuda")
    request = torch.searchsorted(state["tree_start"][1:].long(), node, right=True)
    return request, node - state["tree_start"].long()[request]


def _plain_tree(state):
    words = -(-state["case"]["nodes"] // 32)
    request, local = _owner(state)
    start = state["tree_start"].long()[request]
    bits = torch.zeros((local.numel(), words * 32), dtype=torch.bool, device="cuda")
    bits.scatter_(1, local[:, None], True)
    at, depth = local, torch.zeros_like(local)
    for _ in range(state["deepest"]):
        up = state["parents"].long()[start + at]
        depth = depth + (up >= 0)
        at = torch.where(up >= 0, up, at)
        bits.scatter_(1, at[:, None], True)
    weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    mask = (bits.view(-1, words, 32) * weights).sum(dim=2)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    cached = state.get("cached")
    positions = depth if cached is None else depth + cached.long()[request]
    return {"mask": mask, "positions": positions.to(torch.int32)}


def _plain_attention(state):
    case = state["case"]
    hq, hkv, d, n_max = case["hq"], case["hkv"], case["d"], case["nodes"]
    shift = torch.arange(32, device="cuda")
    at = 0
    for row, n, length in zip(state["row_list"], state["sizes"], state["cached_list"]):
        slots = state["table"][row, : length + n].long()
        k = state["k"][slots].float().transpose(0, 1)  # [hkv, keys, d]
        v = state["v"][slots].float().transpose(0, 1)
        q = state["q"][at : at + n].float().view(n, hkv, hq // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
        s = (q @ k.transpose(1, 2) * state["scale"]).view(hkv, n, hq // hkv, length + n)
        seen = ((state["mask"][at : at + n, :, None] >> shift) & 1).view(n, -1)[:, :n] != 0
        s[..., length:].masked_fill_(~seen[None, :, None, :], -math.inf)
        p = torch.exp(s - s.amax(dim=3, keepdim=True))
        o = (p.view(hkv, -1, length + n) @ v).view(hkv, n, hq // hkv, d) / p.sum(dim=3, keepdim=True)
        state["out"][at : at + n] = o.permute(1, 0, 2, 3).reshape(n, hq * d).to(torch.bfloat16)
        at += n
    return {"out": state["out"]}


def _plain_verify(state):
    """All requests walk their trees in step; in 64 bits, since tokens hang on comparisons of sums."""
    case, probs = state["case"], state["probs"]
    request, local = _owner(state)
    start = state["tree_start"].long()
    count, most = len(state["sizes"]), max(state["sizes"])
    padded = torch.full((count, most), -2, dtype=torch.int64, device="cuda")
    padded[request, local] = state["parents"].long()
    index = torch.arange(most, device="cuda")
    rows = torch.arange(count, device="cuda")
    cur = torch.zeros(count, dtype=torch.int64, device="cuda")
    alive = torch.ones(count, dtype=torch.bool, device="cuda")
    rank = torch.zeros((count, most), dtype=torch.int64, device="cuda") + most + index  # rejected nodes come last
    rank[:, 0] = 0
    accepted = torch.zeros(count, dtype=torch.int64, device="cuda")
    token = torch.zeros(count, dtype=torch.int64, device="cuda")
    for _ in range(state["deepest"] + 1):
        row = start[:-1] + cur
        x = state["logits"][row].double()
        if case["greedy"]:
            r, total = None, None
            best = x.argmax(dim=1)
        else:
            p = torch.exp((x - x.amax(dim=1, keepdim=True)) / TEMPERATURE)
            r = p / p.sum(dim=1, keepdim=True)
            total = r.sum(dim=1)
        found = torch.full((count,), -1, dtype=torch.int64, device="cuda")
        last = torch.zeros(count, dtype=torch.int64, device="cuda")
        for _ in range(state["broadest"]):
            is_child = (padded == cur[:, None]) & (index > last[:, None])
            child = torch.where(is_child, index, most).amin(dim=1)
            is_open = alive & (child < most) & (found < 0)
            node = start[:-1] + child.clamp(max=most - 1)
            node = torch.minimum(node, start[1:] - 1)
            t = state["tokens"][node]
            if case["greedy"]:
                take = is_open & (t == best)
            else:
                q = probs[row, t].double() if probs is not None else 1.0
                take = is_open & (state["accept"][node].double() * q * total < r[rows, t])
            found = torch.where(take, child, found)
            last = torch.where(child < most, child, last)
            lost = is_open & ~take
            if not case["greedy"]:
                if probs is not None:
                    rest = (r / total[:, None] - probs[row].double()).clamp(min=0)
                else:
                    rest = r.clone()
                    rest[rows, t] = 0
                left = rest.sum(dim=1)
                lost = lost & (left > 0)
                r = torch.where(lost[:, None], rest, r)
                total = torch.where(lost, left, total)
        if not case["greedy"]:
            c = r.cumsum(dim=1)
            best = (c <= (state["sample"].double() * total)[:, None]).sum(dim=1)
            last_token = torch.where(r > 0, torch.arange(r.shape[1], device="cuda"), -1).amax(dim=1)
            best = torch.minimum(best, last_token)
        ends = alive & (found < 0)
        token = torch.where(ends, best, token)
        alive = alive & (found >= 0)
        cur = torch.where(alive, found, cur)
        accepted = accepted + alive
        rank[rows, cur] = torch.where(alive, accepted, rank[rows, cur])
    size = start[1:] - start[:-1]
    order = torch.argsort(rank, dim=1)[index[None, :] < size[:, None]]  # places past a tree's end rank last
    return {"accepted": accepted.to(torch.int32), "next_token": token, "order": order.to(torch.int32)}


def _framework(state):
    from aios_b200.kernel import ops

    case = state["case"]
    if case["op"] == "tree":
        mask, positions = ops.draft_tree(state["parents"], state["tree_start"], max_nodes=case["nodes"],
                                         cached_lens=state["cached"])
        return {"mask": mask, "positions": positions}
    if case["op"] == "attention":
        ops.attention_tree(
            q=state["q"], out=state["out"], k_cache=state["k"], v_cache=state["v"], page_table=state["table"],
            row_table=state["rows"], cached_lens=state["cached"], tree_start=state["tree_start"],
            tree_mask=state["mask"], num_qo_heads=case["hq"], num_kv_heads=case["hkv"], head_dim=case["d"],
            scale=state["scale"], max_cached=state["max_cached"],
        )
        return {"out": state["out"]}
    accepted, token, order = ops.verify_draft(
        state["logits"], state["tokens"], state["parents"], state["tree_start"], state["accept"], state["sample"],
        temperature=TEMPERATURE, greedy=case["greedy"], draft_probs=state["probs"],
    )
    return {"accepted": accepted, "next_token": token, "order": order}


def run(state):
    if own:
        return _framework(state)
    return {"tree": _plain_tree, "attention": _plain_attention, "verify": _plain_verify}[state["case"]["op"]](state)


# ---- definitions in 64 bits --------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(state)
    if case["op"] == "attention":
        return _exact_attention(state)
    return _exact_verify(state)


def _exact_tree(state):
    words = -(-state["case"]["nodes"] // 32)
    parents, cached = state["parents"].tolist(), state["cached"].tolist()
    masks, positions = [], []
    at = 0
    for r, n in enumerate(state["sizes"]):
        bits, depth = [], []
        for i in range(n):
            p = parents[at + i]
            bits.append(1 << i | (bits[p] if p >= 0 else 0))
            depth.append(depth[p] + 1 if p >= 0 else 0)
        for b, e in zip(bits, depth):
            row = [(b >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
            masks.append([w - (1 << 32) if w >> 31 else w for w in row])
            positions.append(cached[r] + e)
        at += n
    return {"mask": _ints(masks), "positions": _ints(positions)}


def _exact_attention(state):
    case = state["case"]
    group, d = case["hq"] // case["hkv"], case["d"]
    parents = state["parents"].tolist()
    out = torch.empty(state["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for row, n, length in zip(state["row_list"], state["sizes"], state["cached_list"]):
        slots = state["table"][row, : length + n].long()
        seen = torch.zeros((n, n), dtype=torch.float64)
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, j] = 1
                j = parents[at + j]
        hide = torch.zeros((n, length + n), dtype=torch.float64, device="cuda")
        hide[:, length:] = torch.log(seen).cuda()
        for h in range(case["hkv"]):
            k, v = state["k"][slots, h].double(), state["v"][slots, h].double()
            for g in range(group):
                c = (h * group + g) * d
                s = torch.addmm(hide, state["q"][at : at + n, c : c + d].double(), k.t(), alpha=state["scale"])
                out[at : at + n, c : c + d] = torch.exp(s - torch.logsumexp(s, dim=1, keepdim=True)) @ v
        at += n
    return {"out": out}


def _exact_verify(state):
    case = state["case"]
    starts, parents = state["tree_start"].tolist(), state["parents"].tolist()
    drawn, accept = state["tokens"].tolist(), state["accept"].tolist()
    accepted, tokens, order = [], [], []
    for r, n in enumerate(state["sizes"]):
        s, path = starts[r], [0]
        while True:
            cur = path[-1]
            x = state["logits"][s + cur].double()
            children = [j for j in range(1, n) if parents[s + j] == cur]
            step = None
            if case["greedy"]:
                top = int((x == x.max()).nonzero()[0])
                step = next((j for j in children if drawn[s + j] == top), None)
            else:
                rest = torch.softmax(x / TEMPERATURE, dim=0)
                q = state["probs"][s + cur].double() if case["probs"] else None
                for j in children:
                    t = drawn[s + j]
                    ratio = rest[t] / rest.sum() / (q[t] if q is not None else 1)
                    if float(ratio) > accept[s + j]:
                        step = j
                        break
                    if q is not None:
                        less = torch.relu(rest / rest.sum() - q)
                    else:
                        less = rest * (torch.arange(rest.numel(), device="cuda") != t)
                    if float(less.sum()) > 0:
                        rest = less
            if step is None:
                break
            path.append(step)
        if not case["greedy"]:
            share = torch.cumsum(rest, dim=0) / rest.sum()
            top = int((share > float(state["sample"][r])).nonzero()[0])
        accepted.append(len(path) - 1)
        tokens.append(top)
        order += path + [j for j in range(n) if j not in path]
    return {"accepted": _ints(accepted), "next_token": torch.tensor(tokens).cuda(), "order": _ints(order)}
