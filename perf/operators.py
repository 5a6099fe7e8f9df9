"""Operators of the paged decode step, case by case: attention whose sequences share a prefix, attention with a distance
bias and a prefix mask, and the slot maps and table rows of a step built on the GPU from request lengths.

`own` false: the plain form of each operator in elementary torch operations; true: the framework's operators."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---- cases -------------------------------------------------------------------------------------------------------
def shared(name, groups, members, prefix, suffix, rows, q_heads, kv_heads, head_dim, page, softcap=0.0, window=-1, slope=False):
    return dict(name=name, op="shared", groups=groups, members=members, prefix=prefix, suffix=suffix, rows=rows,
                q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, softcap=softcap, window=window, slope=slope)


def biased(name, batch, rows, cached, q_heads, kv_heads, head_dim, page, softcap=0.0, window=-1, two_way=False):
    return dict(name=name, op="biased", batch=batch, rows=rows, cached=cached, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, softcap=softcap, window=window, two_way=two_way)


def extend(name, batch, new, cached, page, spare):
    return dict(name=name, op="extend", batch=batch, new=new, cached=cached, page=page, spare=spare)


def listed():
    return [
        # four samples of one short prompt, a few tokens in: the smallest step of its kind, latency counts
        shared("shared_few_samples", 1, 4, 512, 32, 1, 32, 8, 128, 128),
        # 32 samples of one prompt of ordinary length
        shared("shared_samples", 1, 32, 2048, 256, 1, 32, 8, 128, 128),
        # a full decode batch behind one long system prompt
        shared("shared_system_prompt", 1, 256, 4096, 1024, 1, 32, 8, 128, 128),
        # questions about two long documents
        shared("shared_documents", 2, 24, 32768, 512, 1, 32, 8, 128, 128),
        # several prompts with a few samples each, four draft rows to verify per sequence, capped scores, small pages
        shared("shared_draft_rows", 6, 11, 1296, 99, 4, 24, 8, 64, 16, 30.0),
        # one conversation's single decode row under a distance bias, one KV head per query head
        biased("biased_decode_one", 1, 1, 700, 16, 16, 128, 16),
        # a decode batch of ragged contexts under a distance bias
        biased("biased_decode", 64, 1, 8192, 32, 8, 128, 128),
        # prompt chunks appended to ragged cached prefixes under a distance bias
        biased("biased_prefill", 4, 1024, 4096, 32, 8, 128, 128),
        # prompts whose opening part is read in both directions, odd lengths, sliding window
        biased("prefix_mask_prefill", 7, 333, 500, 12, 4, 64, 16, 0.0, 400, True),
        # one new token for each request of a decode batch
        extend("extend_decode", 64, 1, 8192, 128, 0),
        # a step that mixes decode rows with prompt chunks, rows padded to a fixed capacity
        extend("extend_mixed", 300, 512, 4000, 16, 1000),
        # the largest decode batch
        extend("extend_large_batch", 4096, 1, 4096, 64, 0),
    ]


def cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(cost(c) for c in listed())
    while True:
        kind = rng.random()
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8])
        head_dim = rng.choice([64, 128, 128, 256])
        page = rng.choice([16, 32, 64, 128])
        softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
        if kind < 0.45:
            groups = rng.choice([1, 1, 2, 3, 7])
            prefix, rows = log(256, 32768), rng.choice([1, 1, 1, 2, 3])
            c = shared("", groups, log(4, 256) // groups + 2, prefix, log(8, 1024) + rows, rows, kv_heads * group, kv_heads,
                       head_dim, page, softcap, rng.choice([-1, -1, -1, log(64, prefix + 64)]), rng.random() < 0.25)
        elif kind < 0.8:
            decode = rng.random() < 0.5
            batch, rows = (log(1, 128), rng.choice([1, 1, 2])) if decode else (log(1, 8), log(33, 1024))
            c = biased("", batch, rows, log(1, 8192), kv_heads * group, kv_heads, head_dim, page, softcap,
                       rng.choice([-1, -1, -1, log(16, 4096)]), not decode and rng.random() < 0.5)
        else:
            decode = rng.random() < 0.5
            c = extend("", log(1, 4096) if decode else log(1, 512), 1 if decode else log(2, 512), log(1, 8192), page,
                       0 if decode else rng.choice([0, log(1, 2000)]))
            if c["batch"] * (c["cached"] + c["new"]) > 64_000_000:
                continue
        del c["name"]
        if cost(c) <= most:
            return c


# ---- lengths: set by the case alone, ragged -------------------------------------------------------------------------
def spread(i, lo, hi):
    """A value of lo..hi for index i, spread over the range; the largest comes first."""
    return hi - (i * 2654435761 >> 7) % (hi - lo + 1) if hi > lo else lo


def shared_lengths(c):
    """Prefix of each group (whole pages) and cached tokens of each sequence (sequence i is in group i % groups)."""
    page = c["page"]
    prefixes = [max(page, spread(g, c["prefix"] - c["prefix"] // 4, c["prefix"]) // page * page) for g in range(c["groups"])]
    return prefixes, [prefixes[i % c["groups"]] + spread(i, 0, c["suffix"] - c["rows"]) for i in range(c["groups"] * c["members"])]


def biased_lengths(c):
    """(cached, new) of each sequence; rows of 1 stay 1, chunks are ragged; the two-way prefix of each sequence."""
    cached = [spread(i, 0, c["cached"]) for i in range(c["batch"])]
    new = [spread(i + 3, max(1, c["rows"] - c["rows"] // 3), c["rows"]) for i in range(c["batch"])]
    return cached, new, [(a + b) * (4 - i % 4) // 4 if c["two_way"] else 0 for i, (a, b) in enumerate(zip(cached, new))]


def extend_lengths(c):
    cached = [spread(i, 0, c["cached"]) for i in range(c["batch"])]
    # every third request of a mixed step is a decode row, every eleventh is idle
    new = [1 if c["new"] == 1 or i % 3 == 1 else 0 if i % 11 == 5 else spread(i + 3, 1, c["new"]) for i in range(c["batch"])]
    return cached, new


def visible(p, window, two_way=0):
    """How many keys a row at position p sees."""
    return max(p + 1, two_way) - (max(0, p - window + 1) if window > 0 else 0)


def work(c):
    if c["op"] == "extend":
        cached, new = extend_lengths(c)
        pages = sum(-(-(a + b) // c["page"]) - -(-a // c["page"]) for a, b in zip(cached, new))
        rows = sum(new)
        # lengths, new, request, one table cell in, next length and row offset out; free pages; location, position, request and table cell per row
        return {"bytes": c["batch"] * (8 + 4 + 4 + 4 + 8 + 4) + pages * 8 + rows * 16 + c["spare"] * 12, "flops": 0}
    d, token = c["head_dim"], c["kv_heads"] * c["head_dim"] * 4
    per_key = (4 * d + (2 if c["op"] == "biased" or c["slope"] else 0)) * c["q_heads"]
    if c["op"] == "shared":
        prefixes, cached = shared_lengths(c)
        new = [c["rows"]] * len(cached)
        starts = [prefixes[i % c["groups"]] for i in range(len(cached))]
        low = lambda i: max(0, cached[i] - c["window"] + 1) if c["window"] > 0 else 0  # noqa: E731
        firsts = [min(low(i) for i in range(g, len(cached), c["groups"])) for g in range(c["groups"])]
        tokens = sum(max(0, p - f) for p, f in zip(prefixes, firsts))
        tokens += sum(a + b - max(s, low(i)) for i, (a, b, s) in enumerate(zip(cached, new, starts)))
        keys = sum(visible(a + r, c["window"]) for a, b in zip(cached, new) for r in range(b))
    else:
        cached, new, two_way = biased_lengths(c)
        tokens = sum(a + b - (max(0, a - c["window"] + 1) if c["window"] > 0 else 0) for a, b in zip(cached, new))
        keys = sum(visible(a + r, c["window"], f) for a, b, f in zip(cached, new, two_way) for r in range(b))
    rows = sum(new)
    return {"bytes": tokens * token + rows * c["q_heads"] * d * 4 + tokens // c["page"] * 4, "flops": keys * per_key}


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    """What the program has before the call: the pool with its table, the queries, and the step's metadata with its plan."""
    if own:
        import gaudirt_b200
    c, gen = case, torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    if c["op"] == "extend":
        return prepare_extend(c, rng)
    page = c["page"]
    if c["op"] == "shared":
        prefixes, cached = shared_lengths(c)
        new, two_way = [c["rows"]] * len(cached), [0] * len(cached)
        starts = [prefixes[i % c["groups"]] for i in range(len(cached))]
    else:
        cached, new, two_way = biased_lengths(c)
        prefixes, starts = [], [0] * len(cached)
    batch, ends = len(cached), [a + b for a, b in zip(cached, new)]
    own_pages = [-(-(e - s) // page) for e, s in zip(ends, starts)]
    blocks = sum(own_pages) + sum(prefixes) // page
    pages = rng.permutation(blocks + blocks // 16 + 1).astype(np.int64)
    slots, context = len(pages) * page, max(ends)
    table = np.full((batch, context), -1, np.int32)
    tokens = lambda ids: (ids[:, None] * page + np.arange(page)).reshape(-1)  # noqa: E731
    at, heads_of = 0, []
    for p in prefixes:
        heads_of.append(tokens(pages[at:at + p // page]))
        at += p // page
    for i in range(batch):
        if starts[i]:
            table[i, :starts[i]] = heads_of[i % c["groups"]]
        table[i, starts[i]:ends[i]] = tokens(pages[at:at + own_pages[i]])[:ends[i] - starts[i]]
        at += own_pages[i]
    requests = np.repeat(np.arange(batch), new)
    positions = np.concatenate([np.arange(a, e) for a, e in zip(cached, ends)])
    rows, d = len(positions), c["head_dim"]
    pool = torch.randn(2, c["kv_heads"], slots, d, generator=gen, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(rows, c["q_heads"] * d, generator=gen, device=DEV).to(torch.bfloat16)
    slopes = None
    if c["op"] == "biased" or c["slope"]:
        slopes = torch.exp2(-8.0 * torch.arange(1, c["q_heads"] + 1, device=DEV, dtype=torch.float32) / c["q_heads"])
    s = dict(case=c, pool=pool, key_pool=pool[0].transpose(0, 1), value_pool=pool[1].transpose(0, 1), q=q, slopes=slopes,
             scale=1.0 / math.sqrt(d), table=torch.from_numpy(table).to(DEV), positions=torch.from_numpy(positions).to(DEV),
             cached=cached, new=new, two_way=two_way, prefixes=prefixes)
    if own:
        table_host, at = torch.from_numpy(table), torch.from_numpy(table[requests, positions])
        md = gaudirt_b200.PagedMetadata(at, torch.from_numpy(requests), torch.from_numpy(positions), table_host, slots)
        if c["op"] == "shared":
            md._share_prefixes_([i % c["groups"] for i in range(batch)], prefixes)
        if any(two_way):
            md._set_prefix_mask_(two_way)
        md.attention_plan_for(c["q_heads"], c["kv_heads"], d, c["window"])
        s["metadata"] = md
    else:
        width = max(new)
        place = np.concatenate([[0], np.cumsum(new)])
        # rows of every sequence side by side (a padded place repeats the sequence's last row), and where each row ended up
        s["padded"] = torch.from_numpy(np.minimum(place[:-1, None] + np.arange(width), place[1:, None] - 1)).to(DEV)
        s["packed"] = torch.from_numpy(requests * width + (np.arange(rows) - place[requests])).to(DEV)
        s["limit"] = torch.from_numpy(np.maximum(positions, np.asarray(two_way)[requests] - 1)).to(DEV)
        if c["op"] == "shared":
            long, tail = max(prefixes), max(e - b for e, b in zip(ends, starts))
            s["prefix_slots"] = torch.from_numpy(np.stack([np.pad(h, (0, long - len(h))) for h in heads_of])).to(DEV)
            s["tail_slots"] = torch.from_numpy(np.stack([np.pad(table[i, b:e], (0, tail - (e - b))) for i, (b, e) in enumerate(zip(starts, ends))])).long().to(DEV)
            s["starts"] = torch.tensor(starts, device=DEV)
    return s


def prepare_extend(c, rng):
    cached, new = extend_lengths(c)
    batch, page = c["batch"], c["page"]
    context = (max(a + b for a, b in zip(cached, new)) + page - 1) // page * page
    held = [-(-a // page) for a in cached]
    fresh = sum(-(-(a + b) // page) - h for a, b, h in zip(cached, new, held))
    order = rng.permutation(batch + batch // 8 + 1)
    ids = torch.from_numpy(rng.permutation(sum(held) + fresh + 17) + 1).to(DEV)     # page 0 holds the padding slot
    first = torch.tensor(np.concatenate([[0], np.cumsum(held)[:-1]]), device=DEV)
    a = torch.tensor(cached, device=DEV)
    place = torch.arange(context, device=DEV)
    index = (first[:, None] + place // page).clamp_(max=len(ids) - 1)
    rows = torch.where(place < a[:, None], ids[index] * page + place % page, -1).to(torch.int32)
    requests = torch.from_numpy(order[:batch].astype(np.int32)).to(DEV)
    mapping = torch.full((len(order), context), -1, dtype=torch.int32, device=DEV)
    mapping[requests.long()] = rows
    return dict(case=c, mapping=mapping, requests=requests, lengths=a, new=torch.tensor(new, dtype=torch.int32, device=DEV),
                free_pages=ids[sum(held):].contiguous(), used=torch.tensor([5], device=DEV), rows=sum(new) + c["spare"])


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    if state["case"]["op"] == "extend":
        return run_extend(state)
    c = state["case"]
    if own:
        if state["slopes"] is not None:
            return torch.ops.gaudirt._paged_attn_biased(state["q"], None, None, state["key_pool"], state["value_pool"],
                                                        state["metadata"], state["slopes"], c["head_dim"], state["scale"],
                                                        c["softcap"], c["window"])
        return torch.ops.gaudirt._paged_attn_stored(state["q"], state["key_pool"], state["value_pool"], state["metadata"],
                                                    c["head_dim"], state["scale"], c["softcap"], c["window"])
    return plain_shared(state) if c["op"] == "shared" else plain_biased(state)


def run_extend(s):
    if own:
        return torch.ops.gaudirt._extend_paged_requests(s["mapping"], s["requests"], s["lengths"], s["new"], s["free_pages"],
                                                        s["used"], s["case"]["page"], s["rows"]) + (s["mapping"],)
    page, lengths, new, table = s["case"]["page"], s["lengths"], s["new"].long(), s["mapping"]
    ends = torch.cumsum(new, 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    row = torch.arange(s["rows"], device=DEV)
    kept = row < ends[-1]
    row = torch.minimum(row, ends[-1] - 1)                   # rows past the last one repeat it, and are blanked at the end
    which = torch.searchsorted(ends, row, right=True)
    j, start, request = row - offsets[which], lengths[which], s["requests"].long()[which]
    held = (lengths + page - 1) // page
    fresh = (lengths + new + page - 1) // page - held
    first = s["used"] + torch.cumsum(fresh, 0) - fresh
    k = j - (held * page - lengths)[which]                   # tokens past the open page
    position = start + j
    slot = torch.where(k < 0, table[request, (start - 1).clamp(min=0)] + 1 + j,
                       s["free_pages"][(first[which] + torch.div(k, page, rounding_mode="floor")).clamp(min=0, max=len(s["free_pages"]) - 1)] * page + k % page)
    table[request, position] = slot.to(torch.int32)
    blank = lambda v: torch.where(kept, v, -1).to(torch.int32)  # noqa: E731
    return blank(slot), blank(position), blank(request), offsets.to(torch.int32), lengths + new, s["used"] + fresh.sum(), table


def plain_scores(s, raw, distance, seen):
    """Scores of [.., kv head, group, row, key] raw products: scale, cap, bias, mask; `distance`, `seen` [.., row, key]."""
    c = s["case"]
    x = raw * s["scale"]
    if c["softcap"] > 0:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(c["kv_heads"], -1, 1, 1) * distance[..., None, None, :, :].abs().float()
    return x.masked_fill(~seen[..., None, None, :, :], float("-inf"))


def plain_seen(c, limit, position, key):
    seen = key <= limit[..., :, None]
    return seen & (key > position[..., :, None] - c["window"]) if c["window"] > 0 else seen


def plain_biased(s):
    c, d, h = s["case"], s["case"]["head_dim"], s["case"]["kv_heads"]
    batch, width = s["padded"].shape
    q = s["q"][s["padded"]].float().view(batch, width, h, -1, d).permute(0, 2, 3, 1, 4)        # [b, h, g, n, d]
    slots = s["table"].long().clamp(min=0)
    keys, values = (s["pool"][i][:, slots].transpose(0, 1).float() for i in (0, 1))            # [b, h, context, d]
    key = torch.arange(slots.shape[1], device=DEV)
    position, limit = s["positions"][s["padded"]], s["limit"][s["padded"]]
    raw = (q.flatten(2, 3) @ keys.transpose(2, 3)).view(batch, h, -1, width, len(key))
    x = plain_scores(s, raw, position[..., None] - key, plain_seen(c, limit, position, key))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    out = (e.flatten(2, 3) @ values).view(batch, h, -1, width, d) / e.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(batch * width, -1)[s["packed"]].to(torch.bfloat16)


def plain_shared(s):
    c, d, h = s["case"], s["case"]["head_dim"], s["case"]["kv_heads"]
    g, m, n = c["groups"], c["members"], c["rows"]
    q = s["q"].float().view(m, g, n, h, -1, d).permute(1, 0, 3, 4, 2, 5)                       # [g, m, h, group, n, d]
    at = s["positions"].view(m, g, n).permute(1, 0, 2)                                         # [g, m, n]
    starts = s["starts"].view(m, g).t()
    fetch = lambda i, slots: s["pool"][i][:, slots].float()  # noqa: E731
    together = lambda x: x.transpose(1, 2).flatten(2, 4)  # noqa: E731  [g, m, h, group, n, .] -> [g, h, m group n, .]
    apart = lambda x: x.unflatten(2, (m, -1, n)).transpose(1, 2)  # noqa: E731
    # the prefix: one product for all rows of a group
    key = torch.arange(s["prefix_slots"].shape[1], device=DEV)
    seen = (key < starts[..., None, None]) & plain_seen(c, at, at, key)
    raw = together(q) @ fetch(0, s["prefix_slots"]).transpose(0, 1).transpose(2, 3)
    x1 = plain_scores(s, apart(raw), at[..., None] - key, seen)
    # what every sequence has of its own
    tails = s["tail_slots"].view(m, g, -1).transpose(0, 1)
    key = starts[..., None, None] + torch.arange(tails.shape[2], device=DEV)                  # [g, m, 1, tail]
    k2, v2 = (fetch(i, tails).permute(1, 2, 0, 3, 4) for i in (0, 1))                          # [g, m, h, tail, d]
    raw = (q.flatten(3, 4) @ k2.transpose(3, 4)).unflatten(3, (-1, n))
    x2 = plain_scores(s, raw, at[..., None] - key, plain_seen(c, at, at, key))
    top = torch.maximum(x1.amax(-1, keepdim=True), x2.amax(-1, keepdim=True))
    e1, e2 = torch.exp(x1 - top), torch.exp(x2 - top)
    out = apart(together(e1) @ fetch(1, s["prefix_slots"]).transpose(0, 1)) + (e2.flatten(3, 4) @ v2).unflatten(3, (-1, n))
    out = out / (e1.sum(-1, keepdim=True) + e2.sum(-1, keepdim=True))
    return out.permute(1, 0, 4, 2, 3, 5).reshape(m * g * n, -1).to(torch.bfloat16)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "extend":
        page, free, used = s["case"]["page"], s["free_pages"].tolist(), int(s["used"])
        table, lengths, new, requests = s["mapping"].cpu().numpy(), s["lengths"].tolist(), s["new"].tolist(), s["requests"].tolist()
        rows, offsets = [], [0]
        for a, n, r in zip(lengths, new, requests):
            for p in range(a, a + n):
                if p % page:
                    slot = int(table[r, p - 1]) + 1
                else:
                    slot = free[used] * page
                    used += 1
                table[r, p] = slot
                rows.append((slot, p, r))
            offsets.append(len(rows))
        rows += [(-1, -1, -1)] * (s["rows"] - len(rows))
        columns = [torch.tensor(x, dtype=torch.int32) for x in zip(*rows)]
        return (*columns, torch.tensor(offsets, dtype=torch.int32), torch.tensor([a + n for a, n in zip(lengths, new)]),
                torch.tensor([used]), torch.from_numpy(table))
    c, d = case, case["head_dim"]
    share = c["q_heads"] // c["kv_heads"]
    out, first = [], 0
    for i, (a, b) in enumerate(zip(s["cached"], s["new"])):
        slots = s["table"][i, :a + b].long()
        k, v = (s["pool"][x][:, slots].double().repeat_interleave(share, 0) for x in (0, 1))
        q = s["q"][first:first + b].double().view(b, c["q_heads"], d)
        x = torch.einsum("rhd,hkd->hrk", q, k) / math.sqrt(d)
        if c["softcap"] > 0:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        p, j = torch.arange(a, a + b, device=DEV)[:, None], torch.arange(a + b, device=DEV)[None, :]
        if s["slopes"] is not None:
            x = x - s["slopes"].double()[:, None, None] * (p - j).abs()
        hidden = (j > p) & (j >= s["two_way"][i])
        if c["window"] > 0:
            hidden = hidden | (j <= p - c["window"])
        x = x.masked_fill(hidden, float("-inf"))
        weight = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
        out.append(torch.einsum("hrk,hkd->rhd", weight, v).reshape(b, -1))
        first += b
    return torch.cat(out)
