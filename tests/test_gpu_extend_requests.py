"""Slot maps and table rows built on the device from request lengths: every output against a loop over the requests, the
batches that are refused whole, and the step as it is used (extend, validate, store, attend)."""
import pytest
import torch

from tests import steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def rt():
    import gaudirt_b200
    gaudirt_b200._C._take_device_status()
    return gaudirt_b200


def make(cached, new, page, spare_requests=3, spare_pages=2, used=1, seed=0):
    gen = torch.Generator().manual_seed(seed)
    batch = len(cached)
    context = max(a + b for a, b in zip(cached, new)) + 1
    held = [-(-c // page) for c in cached]
    fresh = [-(-(c + n) // page) - h for c, n, h in zip(cached, new, held)]
    ids = torch.randperm(sum(held) + sum(fresh) + used + spare_pages, generator=gen) + 1
    requests = torch.randperm(batch + spare_requests, generator=gen)[:batch].to(torch.int32)
    table = torch.full((batch + spare_requests, context), -1, dtype=torch.int32)
    at = 0
    for r, c, h in zip(requests.tolist(), cached, held):
        slots = (ids[at:at + h, None] * page + torch.arange(page)).reshape(-1)[:c]
        table[r, :c] = slots.to(torch.int32)
        at += h
    return dict(mapping=table, batch_requests=requests, lengths=torch.tensor(cached),
                new_tokens=torch.tensor(new, dtype=torch.int32), free_pages=ids[sum(held):].contiguous(),
                used_pages=torch.tensor([used]), page_size=page)


def expected(a, rows):
    table, page, used = a["mapping"].clone(), a["page_size"], int(a["used_pages"])
    free, out, offsets = a["free_pages"].tolist(), [], [0]
    for r, c, n in zip(a["batch_requests"].tolist(), a["lengths"].tolist(), a["new_tokens"].tolist()):
        for p in range(c, c + n):
            if p % page:
                slot = int(table[r, p - 1]) + 1
            else:
                slot, used = free[used] * page, used + 1
            table[r, p] = slot
            out.append((slot, p, r))
        offsets.append(len(out))
    out += [(-1, -1, -1)] * (rows - len(out))
    columns = [torch.tensor(x, dtype=torch.int32) for x in zip(*out)]
    return (*columns, torch.tensor(offsets, dtype=torch.int32), a["lengths"] + a["new_tokens"], torch.tensor([used])), table


def call(a, rows):
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    return torch.ops.gaudirt._extend_paged_requests(**on, rows=rows), on


def spread(n, hi, seed):
    return torch.randint(0, hi + 1, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


CASES = {
    "one_new": ([0], [1], 16),
    "one_in_open_page": ([5], [1], 16),
    "page_ends": ([16, 15, 17, 0, 31, 32], [1, 1, 1, 16, 2, 33], 16),
    "page_of_one": ([3, 0, 7], [4, 1, 0], 1),
    "page_of_three": ([3, 1, 8, 0], [4, 7, 0, 2], 3),
    "idle_first_and_last": ([4, 9, 2, 8], [0, 3, 0, 0], 8),
    "nothing_new": ([4, 9], [0, 0], 8),
    "ragged": (spread(100, 300, 1), spread(100, 70, 2), 32),
    "warp_edge": (spread(33, 50, 3), spread(33, 5, 4), 8),
    "cta_edge": (spread(1024, 40, 5), spread(1024, 3, 6), 16),
    "past_cta_edge": (spread(1025, 40, 7), spread(1025, 3, 8), 16),
    "largest_one_launch": (spread(4096, 20, 9), [1] * 4096, 8),
    "two_launches": (spread(4097, 20, 9), spread(4097, 2, 10), 8),
    "largest": (spread(65536, 9, 11), spread(65536, 1, 12), 4),
}


@pytest.mark.parametrize("spare", [0, 1, 100])
@pytest.mark.parametrize("case", CASES)
def test_against_a_loop_over_the_requests(rt, case, spare):
    cached, new, page = CASES[case]
    a = make(cached, new, page, seed=len(case))
    rows = max(1, sum(new) + spare)
    want, table = expected(a, rows)
    got, on = call(a, rows)
    for name, g, w in zip(("locations", "positions", "row_requests", "row_offsets", "next_lengths", "next_used"), got, want):
        assert g.dtype == w.dtype and torch.equal(g.cpu(), w), name
    assert torch.equal(on["mapping"].cpu(), table)
    for name in ("batch_requests", "lengths", "new_tokens", "free_pages", "used_pages"):
        assert torch.equal(on[name].cpu(), a[name]), name
    assert rt._C._take_device_status() == 0


def test_table_wider_than_its_rows(rt):
    a = make([5, 40], [30, 2], 16)
    wide = torch.full((a["mapping"].size(0), a["mapping"].size(1) + 13), 77, dtype=torch.int32, device=DEV)
    view = wide[:, 5:5 + a["mapping"].size(1)]
    view.copy_(a["mapping"])
    want, table = expected(a, 32)
    got = torch.ops.gaudirt._extend_paged_requests(view, *(a[k].to(DEV) for k in ("batch_requests", "lengths", "new_tokens",
                                                                                 "free_pages", "used_pages")), 16, 32)
    assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want)) and torch.equal(view.cpu(), table)
    assert (wide[:, :5] == 77).all() and (wide[:, 5 + a["mapping"].size(1):] == 77).all()


FAULTS = {
    "length_negative": lambda a: a["lengths"].__setitem__(1, -1),
    "length_past_table": lambda a: a["lengths"].__setitem__(1, a["mapping"].size(1)),
    "length_huge": lambda a: a["lengths"].__setitem__(1, 2**62),
    "new_negative": lambda a: a["new_tokens"].__setitem__(0, -1),
    "new_huge": lambda a: a["new_tokens"].__setitem__(0, 2**31 - 1),
    "request_negative": lambda a: a["batch_requests"].__setitem__(2, -1),
    "request_past_table": lambda a: a["batch_requests"].__setitem__(2, a["mapping"].size(0)),
    "request_twice": lambda a: a["batch_requests"].__setitem__(2, int(a["batch_requests"][0])),
    "used_negative": lambda a: a["used_pages"].__setitem__(0, -1),
    "used_past_list": lambda a: a["used_pages"].__setitem__(0, 10**6),
    "too_few_pages": lambda a: a["used_pages"].__setitem__(0, int(a["used_pages"][0]) + 3),
}


@pytest.mark.parametrize("batch", [5, 5000])
@pytest.mark.parametrize("fault", FAULTS)
def test_refused_batches_change_nothing(rt, fault, batch):
    a = make(spread(batch, 30, 1), [3] * batch, 8, seed=2)
    FAULTS[fault](a)
    got, on = call(a, 3 * batch)
    assert rt._C._take_device_status() == 8                   # GK_DEV_BAD_METADATA
    for g in got[:3]:
        assert (g == -1).all()
    assert (got[3] == 0).all() and torch.equal(got[4].cpu(), a["lengths"]) and torch.equal(got[5].cpu(), a["used_pages"])
    assert torch.equal(on["mapping"].cpu(), a["mapping"])


def test_more_tokens_than_rows(rt):
    a = make([3, 4], [5, 6], 4)
    got, on = call(a, 10)
    assert rt._C._take_device_status() == 8 and (got[0] == -1).all() and torch.equal(on["mapping"].cpu(), a["mapping"])


def test_impossible_pages_and_slots_are_left_out(rt):
    a = make([8, 3, 5], [2, 2, 1], 8, used=0)
    a["free_pages"][0] = 2**40                                # the first request's fresh page does not fit a slot
    a["mapping"][a["batch_requests"][1].long(), 2] = -1       # the second one's last cached token has no slot
    got, on = call(a, 5)
    assert rt._C._take_device_status() == 3                   # GK_DEV_BAD_SLOT | GK_DEV_BAD_TABLE
    assert got[0].tolist()[:4] == [-1] * 4 and got[0][4] >= 0
    assert got[1].tolist() == [8, 9, 3, 4, 5]


def test_captured_decode_loop(rt):
    """One captured launch replayed as the lengths grow: the outputs feed the next step in place."""
    a = make([14, 0, 30], [1, 1, 1], 16, spare_pages=12)
    a["mapping"] = torch.nn.functional.pad(a["mapping"], (0, 40), value=-1)
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    graph = torch.cuda.CUDAGraph()
    first = torch.ops.gaudirt._extend_paged_requests(**{**on, "mapping": on["mapping"].clone()}, rows=3)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = torch.ops.gaudirt._extend_paged_requests(**on, rows=3)
        on["lengths"].copy_(out[4])
        on["used_pages"].copy_(out[5])
    for turn in range(20):
        want, table = expected(a, 3)
        graph.replay()
        assert all(torch.equal(g.cpu(), w) for g, w in zip(out, want)) and torch.equal(on["mapping"].cpu(), table)
        if turn == 0:
            assert all(torch.equal(f.cpu(), w) for f, w in zip(first, want))
        a["mapping"], a["lengths"], a["used_pages"] = table, want[4], want[5]
    assert rt._C._take_device_status() == 0


def test_argument_checks(rt):
    a = make([3, 4], [5, 6], 4)
    on = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    call_ = torch.ops.gaudirt._extend_paged_requests
    for change, message in (({"lengths": on["lengths"].int()}, "int64 indices"), ({"free_pages": on["free_pages"].int()}, "int64 indices"),
                            ({"used_pages": on["used_pages"].repeat(2)}, "used count"), ({"new_tokens": on["new_tokens"].long()}, "int32 request ids"),
                            ({"batch_requests": on["batch_requests"][:1]}, "int32 request ids"), ({"mapping": on["mapping"].long()}, "int32 request map"),
                            ({"mapping": on["mapping"].t()}, "int32 request map"), ({"mapping": on["mapping"][:1].expand(5, -1)}, "int32 request map"),
                            ({"page_size": 0}, "unsupported page size"), ({"rows": 0}, "unsupported page size")):
        with pytest.raises(RuntimeError, match=message):
            call_(**{**on, "rows": 11, **change})
    with pytest.raises(RuntimeError):
        call_(**{**on, "rows": 11, "lengths": a["lengths"]})


def test_extend_validate_store_attend(rt):
    """The step as a scheduler runs it: slots and index vectors from device lengths, validated metadata over them, sequences
    that share a prefix, rotated rows stored, biased attention over the pool."""
    prefix, page, heads, kv_heads, d = 96, 16, 8, 2, 128
    step = steps.shared_step([prefix], [(0, 21, 1), (0, 0, 1), (-1, 40, 1), (0, 64, 2)], heads, kv_heads, d, page, seed=6)
    table = step.mapping.clone()
    fresh = []
    for i, (c, n) in enumerate(zip(step.cached, step.lengths)):     # take the new rows' cells out again
        for p in range(c, c + n):
            if p % page == 0:
                fresh.append(int(table[i, p]) // page)
            table[i, p] = -1
    table = table.to(DEV)
    batch = torch.arange(len(step.cached), dtype=torch.int32, device=DEV)
    locations, positions, requests, offsets, lengths, used = rt._C._extend_paged_requests(
        table, batch, torch.tensor(step.cached, device=DEV), torch.tensor(step.lengths, dtype=torch.int32, device=DEV),
        torch.tensor(fresh, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV), page, len(step.positions))
    assert torch.equal(table.cpu(), step.mapping) and torch.equal(locations.cpu(), step.locations)
    assert torch.equal(requests.cpu().long(), step.requests) and int(used) == len(fresh)
    md = rt.PagedMetadata.from_device(locations, batch, positions, table, step.cached, step.lengths, step.slots)
    md._share_prefixes_(step.groups, step.prefixes)
    md._set_prefix_sharing(1, 0)
    pool = step.pool.to(DEV)
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    angle = torch.arange(step.mapping.size(1))[:, None] / 10000 ** (torch.arange(d // 2) / (d // 2))
    cache = torch.cat([angle.cos(), angle.sin()], 1).to(torch.bfloat16).to(DEV)
    slopes = steps.slopes_of(heads)
    q = torch.ops.gaudirt._rotary_kv_store(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), cache, md, kp, vp, d, d, True)
    out = torch.ops.gaudirt._paged_attn_biased(q, None, None, kp, vp, md, slopes.to(DEV), d, step.scale)
    step.q = q.cpu()
    steps.check(out, *steps.attend64(step, pool.cpu(), slopes=slopes))
    assert rt._C._take_device_status() == 0
