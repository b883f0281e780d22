"""Plain 64-bit restatements of the drafted trees' operators, on the CPU or the GPU."""

from __future__ import annotations

import random

import torch


def trees(sizes: list[int], kind: str, seed: int = 0) -> list[list[int]]:
    """Parents of trees of these sizes: a "chain", a "star", or "mixed"."""
    rng = random.Random(seed)
    out = []
    for n in sizes:
        if kind == "chain":
            p = [i - 1 for i in range(n)]
        elif kind == "star":
            p = [-1 if i == 0 else 0 for i in range(n)]
        else:
            p = [-1 if i == 0 else rng.randint(max(0, i - 6), i - 1) for i in range(n)]
        out.append(p)
    return out


def starts(sizes: list[int]) -> list[int]:
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def tree_bits(parents: list[list[int]], words: int, cached: list[int] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    masks, positions = [], []
    for r, ps in enumerate(parents):
        for i in range(len(ps)):
            row, j, depth = [0] * words, i, -1
            while j >= 0:
                row[j // 32] |= 1 << (j % 32)
                j, depth = ps[j], depth + 1
            masks.append([w - (1 << 32) if w >> 31 else w for w in row])
            positions.append((cached[r] if cached else 0) + depth)
    return torch.tensor(masks, dtype=torch.int32).reshape(-1, words), torch.tensor(positions, dtype=torch.int32)


def attention(q, k, v, table, rows, cached, sizes, mask, hq, hkv, d, scale):
    """(o, sum p |v|, largest sum |q_e k_e| scale) in fp64; mask bits past a tree's size are ignored."""
    group = hq // hkv
    out = torch.zeros(q.shape[0], hq, d, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    top = 0.0
    shift = torch.arange(32, device=q.device)
    at = 0
    for row, n, length in zip(rows, sizes, cached):
        if n == 0:
            continue
        slots = table[row, : length + n].long()
        seen = torch.ones(n, length + n, dtype=torch.bool, device=q.device)
        own = ((mask[at : at + n, :, None].long() >> shift) & 1).reshape(n, -1)[:, :n] != 0
        seen[:, length : length + own.shape[1]] = own
        seen[:, length + own.shape[1] :] = False
        for h in range(hq):
            kk, vv = k[slots, h // group].double(), v[slots, h // group].double()
            qq = q[at : at + n].double().view(n, hq, d)[:, h]
            s = (qq @ kk.t() * scale).masked_fill(~seen, -float("inf"))
            m = s.amax(dim=1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m)).masked_fill(~seen, 0)
            total = p.sum(dim=1, keepdim=True)
            p = torch.where(total > 0, p / total, p)
            clean = seen.any(dim=0)
            out[at : at + n, h] = p[:, clean] @ vv[clean]
            mag[at : at + n, h] = p[:, clean] @ vv[clean].abs()
            if bool(clean.any()):
                top = max(top, float((qq.abs() @ kk[clean].abs().t()).max()) * abs(scale))
        at += n
    return out.view(q.shape[0], hq * d), mag.view(q.shape[0], hq * d), top


def attention_tolerance(out, mag, top, keys: int, d: int):
    """Weights are rounded to bf16 (2^-8 of each), the result as well. Scores are fp32 sums of d products
    (2^-23 of the magnitudes a term), scaled: their error is a relative one of each weight, and of the sum;
    2^-21 a chunk of 64 keys covers the exponentials and rescalings, and the sums of weights."""
    delta = 2 * (d + 4) * 2.0**-23 * top + (keys / 64 + 4) * 2.0**-21
    return (2.0**-8 + 2 * delta) * mag * (1 + 2.0**-8) + 2.0**-8 * out.abs() + 1e-30


def verify(logits, tokens, parents, accept, sample, temperature=1.0, greedy=False, probs=None):
    """Per tree, in fp64: (accepted, next token, order) as lists."""
    accepted, following, order = [], [], []
    at = 0
    for r, ps in enumerate(parents):
        n = len(ps)
        if n == 0:
            accepted.append(0)
            following.append(-1)
            continue
        path, token = [0], None
        while token is None:
            cur = path[-1]
            x = logits[at + cur].double()
            top = float(x.max())
            if top != top or top == -float("inf") or (not greedy and top == float("inf")):
                token = -1
                break
            children = [j for j in range(cur + 1, n) if ps[j] == cur]
            found = None
            if greedy:
                best = int((x == top).nonzero()[0])
                found = next((j for j in children if int(tokens[at + j]) == best), None)
            else:
                rest = torch.exp((x - top) / temperature)
                rest = rest / rest.sum()
                for j in children:
                    t = int(tokens[at + j])
                    if not 0 <= t < x.numel():
                        continue
                    q = probs[at + cur].double() if probs is not None else None
                    qx = float(q[t]) if q is not None else 1.0
                    if float(accept[at + j]) * qx * float(rest.sum()) < float(rest[t]):
                        found = j
                        break
                    if q is not None:
                        less = (rest / rest.sum() - q).clamp(min=0)
                    else:
                        less = rest.clone()
                        less[t] = 0
                    if float(less.sum()) > 0:
                        rest = less
                best = None
            if found is not None:
                path.append(found)
            elif greedy:
                token = best
            else:
                c = rest.cumsum(0)
                past = (c > float(sample[r]) * float(c[-1])).nonzero()
                token = int(past[0]) if past.numel() else int((rest > 0).nonzero()[-1])
        accepted.append(len(path) - 1)
        following.append(token)
        order += path + [j for j in range(n) if j not in path]
        at += n
    return accepted, following, order
