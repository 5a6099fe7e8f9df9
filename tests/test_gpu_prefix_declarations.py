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
