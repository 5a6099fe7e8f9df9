"""Attention of sequences that share a prefix: every operator over metadata with declared prefixes against binary64, the
merge of states, and the refusals."""
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


def metadata(rt, step):
    return rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)


def pools(step, stored=False):
    pool = (step.stored_pool() if stored else step.pool).to(DEV)
    return pool, pool[0].transpose(0, 1), pool[1].transpose(0, 1)


def shared_metadata(rt, step, mode=1, pieces=0, splits=0):
    md = metadata(rt, step)
    md._share_prefixes_(step.groups, step.prefixes)
    md._set_prefix_sharing(mode, pieces)
    if splits:
        md._set_split_tokens(splits)
    return md


GEOMETRIES = [(8, 2, 128), (4, 4, 64), (16, 1, 256), (6, 2, 128), (5, 1, 64)]
# name, prefixes, members (group, cached behind the prefix, new rows), page
SHAPES = {
    "two": ([96], [(0, 5, 1), (0, 0, 1)], 16),
    "one_token": ([1], [(0, 3, 1), (0, 0, 1), (0, 70, 1)], 1),
    "odd_page_end": ([37], [(0, 9, 1), (0, 1, 1), (0, 150, 1)], 16),
    "groups_and_others": ([300, 64, 129], [(1, 4, 1), (-1, 33, 1), (0, 0, 1), (2, 17, 1), (0, 140, 1), (-1, 0, 1), (1, 0, 1),
                                          (2, 0, 1), (0, 1, 1)], 32),
    "lone_member": ([128, 256], [(0, 3, 1), (1, 4, 1), (1, 9, 1)], 128),
    "draft_rows": ([257], [(0, 2, 3), (0, 0, 1), (0, 40, 5), (0, 7, 2)], 1),
    "long": ([2048], [(0, 300, 1), (0, 2, 1), (0, 65, 1), (0, 640, 1)], 128),
    "with_chunk": ([200], [(0, 5, 1), (0, 3, 150), (0, 8, 1), (-1, 10, 70)], 8),
}


@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shared_prefix_against_binary64(rt, shape, geometry):
    prefixes, members, page = SHAPES[shape]
    step = steps.shared_step(prefixes, members, *geometry, page, seed=len(shape) + geometry[2])
    md = shared_metadata(rt, step)
    pool, kp, vp = pools(step)
    out = torch.ops.gaudirt.paged_attn(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, step.head_dim, step.scale)
    assert md._last_plan_prefix_records() > 0
    assert torch.equal(pool.cpu().view(torch.int16), step.stored_pool().view(torch.int16))
    steps.check(out, *steps.attend64(step, step.stored_pool()))
    again = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, step.head_dim, step.scale)
    assert torch.equal(out, again)
    assert rt._C._take_device_status() == 0


@pytest.mark.parametrize("pieces", [64, 128, 512, 100000])
@pytest.mark.parametrize("splits", [0, 64])
@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 4, 64), (16, 2, 256)])
def test_any_cut_of_prefix_and_tail(rt, geometry, pieces, splits):
    step = steps.shared_step([777, 130], [(0, 400, 1), (0, 3, 1), (1, 90, 2), (1, 0, 1), (0, 0, 1)], *geometry, 1, seed=5)
    md = shared_metadata(rt, step, pieces=pieces, splits=splits)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, step.head_dim, step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool()))


@pytest.mark.parametrize("geometry,members", [((32, 8, 128), 70), ((16, 1, 64), 40), ((8, 1, 256), 50)])
def test_more_rows_than_one_record_holds(rt, geometry, members):
    step = steps.shared_step([512], [(0, i % 50, 1) for i in range(members)], *geometry, 64, seed=members)
    md = shared_metadata(rt, step)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, step.head_dim, step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool()))


@pytest.mark.parametrize("window", [1, 7, 60, 200, 450, 5000])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 2, 64), (4, 1, 256)])
def test_window_and_softcap(rt, geometry, softcap, window):
    """Windows that end in the tail, reach into the prefix for some rows only, and cover everything."""
    step = steps.shared_step([400], [(0, 100, 1), (0, 0, 1), (0, 20, 3), (0, 250, 1)], *geometry, 16, seed=11)
    md = shared_metadata(rt, step)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, step.head_dim, step.scale, softcap, window)
    steps.check(out, *steps.attend64(step, step.stored_pool(), softcap, window))


@pytest.mark.parametrize("two_way", [False, True])
@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_distance_bias_over_a_shared_prefix(rt, geometry, two_way):
    step = steps.shared_step([300], [(0, 40, 1), (0, 0, 4), (-1, 90, 1), (0, 7, 60), (0, 3, 2)], *geometry, 16, seed=21)
    md = shared_metadata(rt, step)
    if two_way:
        step.two_way = [0, 303, 91, 340, 305]
        md._set_prefix_mask_(step.two_way)
    slopes = steps.slopes_of(step.q_heads)
    _, kp, vp = pools(step)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, slopes.to(DEV),
                                               step.head_dim, step.scale)
    assert md._last_plan_prefix_records() > 0
    steps.check(out, *steps.attend64(step, step.stored_pool(), slopes=slopes))


def test_declared_prefixes_are_used_where_they_pay(rt):
    few = steps.shared_step([64], [(0, 5, 1), (0, 0, 1)], 8, 2, 128, 16, seed=1)
    md = shared_metadata(rt, few, mode=-1)
    md.attention_plan(8, 2, 128)
    assert md._last_plan_prefix_records() == 0
    many = steps.shared_step([8192], [(0, 5, 1)] * 24, 32, 8, 128, 16, seed=1)
    md = shared_metadata(rt, many, mode=-1)
    md.attention_plan(32, 8, 128)
    assert md._last_plan_prefix_records() > 0
    _, kp, vp = pools(many, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(many.q.to(DEV), kp, vp, md, 128, many.scale)
    steps.check(out, *steps.attend64(many, many.stored_pool()))


def test_gathered_destinations(rt):
    """The push form stores the merged rows into every destination's column block."""
    step = steps.shared_step([300], [(0, 40, 1), (0, 0, 1), (-1, 90, 1), (0, 3, 40)], 8, 2, 128, 16, seed=3)
    md = shared_metadata(rt, step)
    plan = md.attention_plan(8, 2, 128)
    _, kp, vp = pools(step)
    width = 8 * 128
    slopes = steps.slopes_of(8)
    for bias in (None, slopes.to(DEV)):
        gathered = [torch.full((len(step.positions), 2 * width), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        torch.ops.gaudirt._paged_attn_push(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md.row_locations(), plan,
                                           [g[:, width:] for g in gathered], 128, step.scale, 0.0, -1, bias)
        for g in gathered:
            assert (g[:, :width] == 7.0).all()
            steps.check(g[:, width:], *steps.attend64(step, step.stored_pool(), slopes=slopes if bias is not None else None))


def test_device_metadata_captured_and_replayed(rt):
    """A step whose index vectors live on the device, captured once and replayed over other requests of the same shape;
    requests that do not share the prefix set the status bit."""
    step = steps.shared_step([160], [(0, 20, 1), (0, 3, 1), (0, 60, 1)], 8, 2, 128, 16, seed=9)
    table = torch.cat([step.mapping, step.mapping.flip(0)]).to(DEV).contiguous()
    table[3:, 160:] = step.mapping[:, 160:].to(DEV)          # requests 3..5: the same prefix, tails in the same order
    table[5, 10] = table[5, 11]                               # request 5 holds another slot inside the prefix
    batch = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    positions, locations = step.positions.to(torch.int32).to(DEV), step.locations.to(DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        md = rt.PagedMetadata.from_device(locations, batch, positions, table, step.cached, step.lengths, step.slots)
        md._share_prefixes_(step.groups, step.prefixes)
        md._set_prefix_sharing(1, 0)
        _, kp, vp = pools(step, stored=True)
        q = step.q.to(DEV)
        eager = torch.ops.gaudirt._paged_attn_stored(q, kp, vp, md, 128, step.scale)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            md._revalidate_(locations, batch, positions)
            out = torch.ops.gaudirt._paged_attn_stored(q, kp, vp, md, 128, step.scale)
        steps.check(eager, *steps.attend64(step, step.stored_pool()))
        for _ in range(2):
            out.zero_()
            graph.replay()
            assert torch.equal(out, eager)
        stream.synchronize()
        assert rt._C._take_device_status() == 0
        batch.copy_(torch.tensor([3, 4, 2], dtype=torch.int32))
        locations.copy_(torch.stack([table[3, step.cached[0]], table[4, step.cached[1]], table[2, step.cached[2]]]))
        graph.replay()
        stream.synchronize()
        assert rt._C._take_device_status() == 0 and torch.equal(out, eager)
        batch.copy_(torch.tensor([0, 1, 5], dtype=torch.int32))
        graph.replay()
        stream.synchronize()
        assert rt._C._take_device_status() & 8               # GK_DEV_BAD_METADATA


def test_other_prefix_is_refused(rt):
    step = steps.shared_step([160], [(0, 20, 1), (0, 3, 1), (-1, 200, 1)], 8, 2, 128, 16, seed=9)
    md = metadata(rt, step)
    with pytest.raises(RuntimeError, match="sequence 2 does not hold"):
        md._share_prefixes_([0, 0, 0], [160])
    with pytest.raises(RuntimeError, match="sequence 1 begins inside"):
        md._share_prefixes_([0, 0, -1], [164])
    with pytest.raises(RuntimeError, match="one group per sequence"):
        md._share_prefixes_([0, 0], [160])
    for groups in ([0, 1, -1], [0, -2, -1]):
        with pytest.raises(RuntimeError, match="group out of range"):
            md._share_prefixes_(groups, [160])
    for prefix in (-1, 10**9):
        with pytest.raises(RuntimeError, match="invalid prefix length"):
            md._share_prefixes_([0, 0, -1], [prefix])
    assert rt._C._take_device_status() == 0
    md._share_prefixes_([0, 0, -1], [160])
    md.attention_plan(8, 2, 128)
    with pytest.raises(RuntimeError, match="already bound"):
        md._share_prefixes_([0, 0, -1], [160])
    with pytest.raises(RuntimeError, match="already bound"):
        md._set_prefix_mask_([0, 0, 0])
    with pytest.raises(RuntimeError, match="sharing mode"):
        md._set_prefix_sharing(2, 0)


def test_prefix_of_no_tokens_and_empty_groups(rt):
    step = steps.shared_step([0, 50, 20], [(0, 20, 1), (0, 3, 1), (2, 0, 1), (2, 1, 1)], 8, 2, 128, 1, seed=4)
    md = shared_metadata(rt, step)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, 128, step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool()))


@pytest.mark.parametrize("geometry", [(8, 2, 128), (6, 2, 64), (8, 1, 256)])
def test_layers_in_a_row_give_the_same_bits(rt, geometry):
    """Prefix, tail and combine of one layer run beside each other and share one split state with the next layer's: many
    layers without a wait in between, the KV store riding in the tail launch, a prefill chunk in the step."""
    step = steps.shared_step([1500, 700], [(0, 30, 1), (1, 400, 1), (0, 0, 1), (-1, 900, 1), (1, 9, 1), (0, 250, 2), (1, 3, 90)],
                             *geometry, 16, seed=17)
    md = shared_metadata(rt, step)
    q, k, v = step.q.to(DEV), step.k.to(DEV), step.v.to(DEV)
    layers = [pools(step) for _ in range(3)]
    for i, (pool, _, _) in enumerate(layers):
        pool.mul_(1.0 - 0.25 * i)
    first = [None] * 3
    for turn in range(60):
        _, kp, vp = layers[turn % 3]
        out = torch.ops.gaudirt.paged_attn(q, k, v, kp, vp, md, step.head_dim, step.scale)
        if first[turn % 3] is None:
            first[turn % 3] = out
        else:
            assert torch.equal(out, first[turn % 3]), turn
    steps.check(first[0], *steps.attend64(step, step.stored_pool()))
    assert rt._C._take_device_status() == 0


def test_everything_at_once(rt):
    """Shared prefixes, a two-way prefix, a distance bias, a cap and a window in one mixed step."""
    step = steps.shared_step([320], [(0, 40, 1), (0, 0, 3), (-1, 90, 1), (0, 100, 1), (0, 7, 80)], 12, 4, 128, 16, seed=23)
    step.two_way = [0, 323, 0, 421, 400]
    md = shared_metadata(rt, step)
    md._set_prefix_mask_(step.two_way)
    slopes = steps.slopes_of(12)
    _, kp, vp = pools(step)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, slopes.to(DEV), 128,
                                               step.scale, 8.0, 300)
    assert md._last_plan_prefix_records() > 0
    steps.check(out, *steps.attend64(step, step.stored_pool(), 8.0, 300, slopes))


@pytest.mark.parametrize("softcap", [0.05, 0.5, 2.0, 1000.0])
def test_caps_from_tight_to_loose(rt, softcap):
    """Scores far inside, around and far outside the cap: both ways of computing it."""
    step = steps.shared_step([300], [(0, 40, 1), (0, 0, 1), (-1, 90, 1)], 8, 2, 128, 16, seed=29)
    md = shared_metadata(rt, step)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, 128, step.scale, softcap)
    steps.check(out, *steps.attend64(step, step.stored_pool(), softcap))


def test_many_short_tails(rt):
    """Enough rows for the form with two warps per tail, of one and of several splits."""
    step = steps.shared_step([256], [(0, (i * 37) % 200, 1) for i in range(130)], 32, 8, 128, 32, seed=31)
    for splits in (0, 64):
        md = shared_metadata(rt, step, splits=splits)
        _, kp, vp = pools(step, stored=True)
        out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, 128, step.scale)
        steps.check(out, *steps.attend64(step, step.stored_pool()))


def test_scheduler_owned_metadata(rt):
    """A table the scheduler vouches for: nothing is compared, the store is a launch of its own."""
    step = steps.shared_step([96], [(0, 21, 1), (0, 0, 1), (0, 64, 2)], 8, 2, 128, 16, seed=6)
    batch = torch.arange(3, dtype=torch.int32, device=DEV)
    md = rt.PagedMetadata._from_scheduler(step.locations.to(DEV), batch, step.positions.to(torch.int32).to(DEV),
                                          step.mapping.to(DEV), step.cached, step.lengths, step.slots, None, 0)
    md._share_prefixes_(step.groups, step.prefixes)
    md._set_prefix_sharing(1, 0)
    pool, kp, vp = pools(step)
    out = torch.ops.gaudirt.paged_attn(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, 128, step.scale)
    assert torch.equal(pool.cpu().view(torch.int16), step.stored_pool().view(torch.int16))
    steps.check(out, *steps.attend64(step, step.stored_pool()))


def test_programmatic_launch_changes_no_bits(rt):
    """The prefix kernel set up while the kernel before it still runs, over several layers."""
    step = steps.shared_step([600], [(0, 30, 1), (0, 0, 1), (-1, 300, 1), (0, 250, 2)], 8, 2, 128, 16, seed=37)
    md = shared_metadata(rt, step)
    pool, kp, vp = pools(step)
    q, k, v = step.q.to(DEV), step.k.to(DEV), step.v.to(DEV)
    call = lambda: torch.ops.gaudirt.paged_attn(q, k, v, kp, vp, md, 128, step.scale)  # noqa: E731
    first = call()
    try:
        assert rt.abi.lib().gk_set_programmatic_launch(1) == 0
        outs = [call() for _ in range(20)]
    finally:
        rt.abi.lib().gk_set_programmatic_launch(0)
    assert all(torch.equal(out, first) for out in outs)
    steps.check(first, *steps.attend64(step, step.stored_pool()))
