"""Steps of sequences that share prefixes, see them in both directions or carry a distance bias, with a binary64 reference
of their attention (CPU tensors, seeded)."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch


@dataclass
class Step:
    q_heads: int
    kv_heads: int
    head_dim: int
    slots: int
    mapping: torch.Tensor        # [sequences, context] int32, -1 where nothing is cached
    requests: torch.Tensor       # [rows]
    positions: torch.Tensor      # [rows]
    locations: torch.Tensor      # [rows]
    cached: list                 # per sequence
    lengths: list                # new rows per sequence
    groups: list                 # per sequence, -1 = none
    prefixes: list               # per group
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    pool: torch.Tensor           # [2, kv_heads, slots, head_dim] before the store
    scale: float
    two_way: list = field(default_factory=list)

    def stored_pool(self):
        pool = self.pool.clone()
        at = self.locations.long()
        pool[0][:, at] = self.k.view(-1, self.kv_heads, self.head_dim).transpose(0, 1)
        pool[1][:, at] = self.v.view(-1, self.kv_heads, self.head_dim).transpose(0, 1)
        return pool


def shared_step(prefixes, members, q_heads, kv_heads, head_dim, page, seed) -> Step:
    """`members`: (group or -1, cached tokens behind the group's prefix, new rows) per sequence.  A prefix is a run of whole
    and partial pages of its own; everything behind it starts on a fresh page's slot with the same offset inside the page."""
    gen = torch.Generator().manual_seed(seed)
    own = [-(-(c + n + (prefixes[g] if g >= 0 else 0) % page) // page) for g, c, n in members]
    heads = [-(-p // page) for p in prefixes]
    count = sum(own) + sum(heads)
    pages = torch.randperm(count + 3, generator=gen)
    slots = (count + 3) * page
    cached = [c + (prefixes[g] if g >= 0 else 0) for g, c, n in members]
    lengths = [n for _, _, n in members]
    context = max(c + n for c, n in zip(cached, lengths)) + 2
    mapping = torch.full((len(members), context), -1, dtype=torch.int32)
    at, prefix_slots = 0, []
    inside = torch.arange(page)
    for p, h in zip(prefixes, heads):
        prefix_slots.append((pages[at:at + h, None] * page + inside).reshape(-1)[:p])
        at += h
    for i, (g, c, n) in enumerate(members):
        start = prefixes[g] if g >= 0 else 0
        if start:
            mapping[i, :start] = prefix_slots[g].to(torch.int32)
        mine = (pages[at:at + own[i], None] * page + inside).reshape(-1)[start % page:]
        mapping[i, start:start + c + n] = mine[:c + n].to(torch.int32)
        at += own[i]
    requests = torch.repeat_interleave(torch.arange(len(members)), torch.tensor(lengths))
    positions = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, lengths)])
    rows = len(positions)
    make = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16)  # noqa: E731
    return Step(q_heads, kv_heads, head_dim, slots, mapping, requests, positions, mapping[requests, positions].contiguous(),
                cached, lengths, [g for g, _, _ in members], list(prefixes), make(rows, q_heads * head_dim),
                make(rows, kv_heads * head_dim), make(rows, kv_heads * head_dim), make(2, kv_heads, slots, head_dim),
                torch.tensor(1.0 / math.sqrt(head_dim), dtype=torch.float32).item(), [0] * len(members))


def plain_step(cached, lengths, q_heads, kv_heads, head_dim, page, seed, two_way=None) -> Step:
    step = shared_step([], [(-1, c, n) for c, n in zip(cached, lengths)], q_heads, kv_heads, head_dim, page, seed)
    if two_way is not None:
        step.two_way = list(two_way)
    return step


def attend64(step: Step, pool, softcap=0.0, window=-1, slopes=None):
    """(out, weighted |v|) in binary64: row at p sees j <= max(p, two_way - 1), j > p - window; the capped score loses
    slope * |p - j|."""
    d, share = step.head_dim, step.q_heads // step.kv_heads
    out, size, first = [], [], 0
    for i, (c, n) in enumerate(zip(step.cached, step.lengths)):
        end = c + n
        at = step.mapping[i, :end].long()
        k, v = (pool[x][:, at].double().repeat_interleave(share, 0) for x in (0, 1))
        q = step.q[first:first + n].double().view(n, step.q_heads, d).transpose(0, 1)
        s = (q @ k.transpose(1, 2)) * step.scale
        if softcap > 0:
            s = softcap * torch.tanh(s / softcap)
        p, j = torch.arange(c, end)[:, None], torch.arange(end)[None, :]
        if slopes is not None:
            s = s - slopes.double()[:, None, None] * (p - j).abs()
        seen = j <= torch.clamp(p, min=step.two_way[i] - 1)
        if window > 0:
            seen = seen & (j > p - window)
        w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        out.append((w @ v).transpose(0, 1).reshape(n, -1))
        size.append((w @ v.abs()).transpose(0, 1).reshape(n, -1))
        first += n
    return torch.cat(out), torch.cat(size)


def check(actual, expected, size):
    """Roundings on the way to a result: every probability once to bf16 (at most 2^-8 of itself, so 2^-8 of the weighted
    |v|) and the result once (2^-8 of itself).  Everything else is fp32: a score of 256 products of unit normals is off by
    at most 256 * 2^-24 * 256 * 0.64 / 16 = 1.6e-4, as much again through the sum of the probabilities, together less than
    2^-11 of the weighted |v| -- an eighth of a bf16 half step on top of each term."""
    got = actual.detach().cpu().double()
    assert torch.isfinite(got).all()
    bound = (size + expected.abs()) * (2.0 ** -8 * 1.125)
    worst = ((got - expected).abs() / bound.clamp(min=1e-30)).max().item()
    assert worst <= 1.0, f"{worst:.3f} of the bound"
    return worst


def slopes_of(q_heads):
    return torch.exp2(-8.0 * torch.arange(1, q_heads + 1, dtype=torch.float32) / q_heads)
