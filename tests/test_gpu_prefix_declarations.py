"""Declarations of shared prefixes that are refused, made again, or not worth following."""
import pytest
import torch

from tests import steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BAD_METADATA = 8


@pytest.fixture(scope="module")
def rt():
    import gaudirt_b200
    gaudirt_b200._C._take_device_status()
    return gaudirt_b200


def device_step(rt):
    """Requests 0 and 1 share 160 tokens, request 2 shares nothing; request 3 has the shape of request 1 and a prefix of its
    own.  The metadata is over requests 0, 1, 2; `swap` puts request 3 in place of request 1."""
    step = steps.shared_step([160], [(0, 20, 1), (0, 3, 1), (-1, 200, 1), (-1, 163, 1)], 8, 2, 128, 16, seed=9)
    table = step.mapping.to(DEV)
    batch = torch.arange(3, dtype=torch.int32, device=DEV)
    positions, locations = step.positions[:3].to(torch.int32).to(DEV), step.locations[:3].to(DEV)
    md = rt.PagedMetadata.from_device(locations, batch, positions, table, step.cached[:3], step.lengths[:3], step.slots)

    def swap():
        batch[1] = 3
        locations[1] = step.locations[3].item()
        md._revalidate_(locations, batch, positions)
        return rt._C._take_device_status()

    return step, md, swap


def test_other_requests_are_judged_by_the_declaration(rt):
    """The two cases that the next test stands between: nothing declared, and declared once."""
    _, md, swap = device_step(rt)
    assert swap() == 0
    _, md, swap = device_step(rt)
    md._share_prefixes_([0, 0, -1], [160])
    assert swap() == BAD_METADATA


@pytest.mark.parametrize("refused", [([0, 0, 0], [160]), ([0, -1, 0], [160]), ([0, 0, -1], [164]), ([0, 0], [160])])
def test_a_refused_declaration_leaves_the_one_before_it_whole(rt, refused):
    step, md, swap = device_step(rt)
    md._share_prefixes_([0, 0, -1], [160])
    with pytest.raises(RuntimeError, match="GaudiRT shared prefix"):
        md._share_prefixes_(*refused)
    md._set_prefix_sharing(1, 0)
    pool = step.stored_pool().to(DEV)
    out = torch.ops.gaudirt._paged_attn_stored(step.q[:3].to(DEV), pool[0].transpose(0, 1), pool[1].transpose(0, 1), md, 128,
                                               step.scale)
    assert md._last_plan_prefix_records() > 0
    expected, size = steps.attend64(step, step.stored_pool())
    steps.check(out, expected[:3], size[:3])
    assert swap() == BAD_METADATA


def test_a_later_declaration_replaces_the_one_before_it(rt):
    _, md, swap = device_step(rt)
    md._share_prefixes_([0, 0, -1], [160])
    md._share_prefixes_([-1, -1, -1], [])
    assert swap() == 0
    _, md, swap = device_step(rt)
    md._share_prefixes_([0, -1, 0], [0])
    md._share_prefixes_([-1, 0, 0], [0])
    md._share_prefixes_([0, 0, -1], [1])
    assert swap() == BAD_METADATA


def test_a_refused_declaration_leaves_other_reports_standing(rt):
    """The status word is the only report of a batch that the slot-map operator refused."""
    _, md, _ = device_step(rt)
    page, one = 16, torch.zeros(1, dtype=torch.int64, device=DEV)
    table = torch.full((2, 32), -1, dtype=torch.int32, device=DEV)
    rt._C._extend_paged_requests(table, torch.tensor([5], dtype=torch.int32, device=DEV), one, torch.ones_like(one).int(), one,
                                 one, page, 1)
    with pytest.raises(RuntimeError, match="sequence 2 does not hold"):
        md._share_prefixes_([0, 0, 0], [160])
    assert rt._C._take_device_status() == BAD_METADATA
    with pytest.raises(RuntimeError, match="sequence 2 does not hold"):
        md._share_prefixes_([0, 0, 0], [160])
    assert rt._C._take_device_status() == 0


def test_a_captured_comparison_outlives_its_declaration(rt):
    """A graph that captured `_revalidate_` writes its verdict on every replay: into memory that is still its own after the
    prefixes were declared anew."""
    step, md, _ = device_step(rt)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        batch = torch.arange(3, dtype=torch.int32, device=DEV)
        positions, locations = step.positions[:3].to(torch.int32).to(DEV), step.locations[:3].to(DEV)
        md = rt.PagedMetadata.from_device(locations, batch, positions, step.mapping.to(DEV), step.cached[:3], step.lengths[:3],
                                          step.slots)
        md._share_prefixes_([0, 0, -1], [160])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            md._revalidate_(locations, batch, positions)
        md._share_prefixes_([-1, -1, -1], [])
        held = [torch.full((4,), 7, dtype=torch.int32, device=DEV) for _ in range(2000)]
        graph.replay()
        stream.synchronize()
        assert all(torch.equal(h, torch.full_like(h, 7)) for h in held)
    assert rt._C._take_device_status() == 0


def draft_metadata(rt, groups, prefixes, behind, rows, page=128):
    """Sequences of `rows` new rows each, `behind` cached tokens behind the prefix of their group."""
    starts = [prefixes[g] if g >= 0 else 0 for g in groups]
    ends = [s + b + rows for s, b in zip(starts, behind)]
    table = torch.full((len(groups), max(ends)), -1, dtype=torch.int32)
    at = 0
    heads = []
    for p in prefixes:
        heads.append(torch.arange(at, at + p, dtype=torch.int32))
        at += -(-p // page) * page
    for i, (g, s, e) in enumerate(zip(groups, starts, ends)):
        if g >= 0:
            table[i, :s] = heads[g]
        table[i, s:e] = torch.arange(at, at + e - s, dtype=torch.int32)
        at += -(-(e - s) // page) * page
    requests = torch.arange(len(groups)).repeat_interleave(rows)
    positions = torch.cat([torch.arange(e - rows, e) for e in ends])
    return rt.PagedMetadata(table[requests, positions].contiguous(), requests, positions, table, at)


# cached tokens behind the prefix, window: nobody sees the prefix; a piece of it that is not worth a launch of its own
@pytest.mark.parametrize("behind,window", [(300, 256), (100, 256), (0, 1)])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_a_window_that_hides_the_prefix_leaves_the_plan_alone(rt, head_dim, behind, window):
    """Short chunks stay where they are when their group is not attended to together: the records are those of a step
    without declarations."""
    plans = []
    for declared in (False, True):
        md = draft_metadata(rt, [0] * 24, [16384], [behind] * 24, 12)
        if declared:
            md._share_prefixes_([0] * 24, [16384])
        plans.append(md.attention_plan_for(32, 8, head_dim, window))
        assert md._last_plan_prefix_records() == 0
    assert torch.equal(*plans)


def test_only_groups_that_are_seen_are_taken_together(rt):
    """Two groups under one window: one sees its prefix and is shared, the other does not and keeps the records it had."""
    groups = [0] * 24 + [1] * 4
    behind = [0] * 24 + [5000] * 4
    md = draft_metadata(rt, groups, [16384, 4096], behind, 12)
    md._share_prefixes_(groups, [16384, 4096])
    md._set_prefix_sharing(1, 0)
    both = md.attention_plan_for(32, 8, 128, 4096)
    assert md._last_plan_prefix_records() > 0
    md = draft_metadata(rt, groups, [16384, 4096], behind, 12)
    md._share_prefixes_([0] * 24 + [-1] * 4, [16384])
    md._set_prefix_sharing(1, 0)
    assert torch.equal(both, md.attention_plan_for(32, 8, 128, 4096))
