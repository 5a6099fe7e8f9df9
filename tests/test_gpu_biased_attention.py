"""Paged attention with a distance bias and with two-way prefixes against binary64, and the refusals."""
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


def metadata(rt, step, splits=0, min_rows=0):
    md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
    if any(step.two_way):
        md._set_prefix_mask_(step.two_way)
    if splits:
        md._set_split_tokens(splits)
    md._set_prefill_min_rows(min_rows)
    return md


def pools(step, stored=False):
    pool = (step.stored_pool() if stored else step.pool).to(DEV)
    return pool, pool[0].transpose(0, 1), pool[1].transpose(0, 1)


GEOMETRIES = [(8, 2, 128), (4, 4, 64), (16, 1, 256), (6, 2, 128), (5, 1, 64)]
# cached and new rows per sequence, page
SHAPES = {
    "one": ([0], [1], 1),
    "decode": ([0, 1, 15, 16, 17, 127, 128, 700], [1] * 8, 16),
    "draft": ([3, 130, 64], [2, 5, 3], 1),
    "chunk": ([0, 100, 37], [200, 64, 333], 8),
    "mixed": ([500, 20, 0, 260], [1, 130, 40, 2], 128),
}


@pytest.mark.parametrize("softcap,window", [(0.0, -1), (4.0, -1), (0.0, 50), (4.0, 130)])
@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("shape", SHAPES)
def test_distance_bias_against_binary64(rt, shape, geometry, softcap, window):
    cached, lengths, page = SHAPES[shape]
    step = steps.plain_step(cached, lengths, *geometry, page, seed=len(shape) + geometry[2])
    slopes = steps.slopes_of(step.q_heads)
    md = metadata(rt, step)
    pool, kp, vp = pools(step)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, slopes.to(DEV),
                                               step.head_dim, step.scale, softcap, window)
    assert torch.equal(pool.cpu().view(torch.int16), step.stored_pool().view(torch.int16))
    steps.check(out, *steps.attend64(step, step.stored_pool(), softcap, window, slopes))
    again = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, md, slopes.to(DEV), step.head_dim,
                                                 step.scale, softcap, window)
    assert torch.equal(out, again)
    assert rt._C._take_device_status() == 0


@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("splits", [64, 4096])
@pytest.mark.parametrize("fused", [0, 1])
def test_bias_under_every_cut_and_staging(rt, splits, fused, form):
    step = steps.plain_step([900, 31, 1500, 0], [1, 2, 1, 1], 8, 2, 128, 16, seed=3)
    slopes = steps.slopes_of(8)
    md = metadata(rt, step, splits=splits, min_rows=-1)
    md._set_fused_combine(fused)
    _, kp, vp = pools(step, stored=True)
    assert rt.abi.lib().gk_set_attention_form(form) == 0
    try:
        out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, md, slopes.to(DEV), 128, step.scale)
    finally:
        rt.abi.lib().gk_set_attention_form(0)
    steps.check(out, *steps.attend64(step, step.stored_pool(), slopes=slopes))


@pytest.mark.parametrize("slopes", [[0.0] * 8, [3.0, 0.0, 0.5, 1e-3, 20.0, 0.25, 1.0, 0.125]])
def test_slopes_from_none_to_steep(rt, slopes):
    step = steps.plain_step([900, 3], [1, 300], 8, 2, 128, 16, seed=8)
    slopes = torch.tensor(slopes)
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, metadata(rt, step), slopes.to(DEV), 128,
                                               step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool(), slopes=slopes))
    if not slopes.any():                                     # the decode row: a bias of nothing changes no bit
        plain = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, metadata(rt, step), 128, step.scale)
        assert torch.equal(plain[:1], out[:1])


# cached, new rows, two-way prefix per sequence
TWO_WAY = {
    "whole_prompt": ([0, 0], [200, 64], [200, 64]),
    "part": ([0, 0, 0, 0], [333, 140, 41, 3], [100, 1, 40, 2]),
    "chunk_behind_prefix": ([128, 500], [150, 2], [128, 30]),
    "prefix_ends_inside": ([100, 90, 300], [260, 37, 4], [359, 100, 302]),
    "one_row": ([0, 5], [1, 1], [1, 6]),
}


@pytest.mark.parametrize("window", [-1, 60])
@pytest.mark.parametrize("min_rows", [0, -1])
@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("shape", TWO_WAY)
def test_two_way_prefix_against_binary64(rt, shape, geometry, min_rows, window):
    """min_rows -1 sends every row through the decode kernel, 0 the chunks through the tensor-core kernel."""
    cached, lengths, two_way = TWO_WAY[shape]
    step = steps.plain_step(cached, lengths, *geometry, 16, seed=len(shape), two_way=two_way)
    md = metadata(rt, step, min_rows=min_rows)
    pool, kp, vp = pools(step)
    out = torch.ops.gaudirt.paged_attn(step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), kp, vp, md, step.head_dim, step.scale,
                                       0.0, window)
    steps.check(out, *steps.attend64(step, step.stored_pool(), 0.0, window))
    slopes = steps.slopes_of(step.q_heads)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, md, slopes.to(DEV), step.head_dim,
                                               step.scale, 6.0, window)
    steps.check(out, *steps.attend64(step, step.stored_pool(), 6.0, window, slopes))


def test_causal_prefix_mask_changes_nothing(rt):
    step = steps.plain_step([100, 3], [1, 300], 8, 2, 128, 16, seed=8)
    md = metadata(rt, step)
    md._set_prefix_mask_([101, 4])                            # nothing that the causal mask does not show already
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, 128, step.scale)
    plain = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, metadata(rt, step), 128, step.scale)
    assert torch.equal(out, plain)


def test_strided_and_offset_inputs(rt):
    """Q, K and V as column slices of one packed projection whose rows are 2-byte aligned only."""
    step = steps.plain_step([70, 0, 12], [1, 90, 2], 8, 2, 64, 16, seed=8)
    slopes = steps.slopes_of(8)
    packed = torch.empty(len(step.positions), 8 * 64 + 2 * 2 * 64 + 1, dtype=torch.bfloat16, device=DEV)[:, 1:]
    q, k, v = packed[:, :512], packed[:, 512:640], packed[:, 640:]
    q.copy_(step.q), k.copy_(step.k), v.copy_(step.v)
    _, kp, vp = pools(step)
    out = torch.ops.gaudirt._paged_attn_biased(q, k, v, kp, vp, metadata(rt, step), slopes.to(DEV), 64, step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool(), slopes=slopes))


def test_refusals(rt):
    step = steps.plain_step([70, 0], [1, 90], 8, 2, 64, 16, seed=8)
    pool, kp, vp = pools(step)
    before = pool.clone()
    q, k, v, slopes = step.q.to(DEV), step.k.to(DEV), step.v.to(DEV), steps.slopes_of(8).to(DEV)
    md = metadata(rt, step)
    call = lambda s, **kw: torch.ops.gaudirt._paged_attn_biased(q, kw.get("k", k), kw.get("v", v), kp, vp, md, s, 64, step.scale)  # noqa: E731
    for bad in (slopes[:7], slopes.double(), slopes.cpu(), slopes.view(2, 4), torch.cat([slopes, slopes])[::2]):
        with pytest.raises(RuntimeError, match="slopes must be"):
            call(bad)
    with pytest.raises(RuntimeError, match="Q/K/V"):
        call(slopes, v=None)
    fresh = lambda: rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)  # noqa: E731
    with pytest.raises(RuntimeError, match="sequence 1 reaches past its last row"):
        fresh()._set_prefix_mask_([0, 91])
    with pytest.raises(RuntimeError, match="sequence 0 reaches past its last row"):
        fresh()._set_prefix_mask_([-1, 0])
    with pytest.raises(RuntimeError, match="one prefix per sequence"):
        fresh()._set_prefix_mask_([0])
    assert torch.equal(pool, before)
    assert rt._C._take_device_status() == 0


def test_same_bits_on_every_launch(rt):
    step = steps.plain_step([500, 20, 0, 260], [1, 330, 140, 2], 8, 2, 128, 16, seed=41, two_way=[0, 200, 140, 0])
    slopes = steps.slopes_of(8).to(DEV)
    md = metadata(rt, step)
    _, kp, vp = pools(step, stored=True)
    call = lambda: torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, md, slopes, 128, step.scale)  # noqa: E731
    first = call()
    assert all(torch.equal(call(), first) for _ in range(20))


def test_rising_bias(rt):
    """Negative slopes: the farthest keys weigh most."""
    step = steps.plain_step([300, 3], [1, 200], 8, 2, 128, 16, seed=43)
    slopes = -steps.slopes_of(8) / 16
    _, kp, vp = pools(step, stored=True)
    out = torch.ops.gaudirt._paged_attn_biased(step.q.to(DEV), None, None, kp, vp, metadata(rt, step), slopes.to(DEV), 128,
                                               step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool(), slopes=slopes))


def test_captured_and_replayed(rt):
    step = steps.plain_step([70, 0, 12], [1, 90, 2], 8, 2, 64, 16, seed=8, two_way=[0, 50, 0])
    slopes = steps.slopes_of(8).to(DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        md = metadata(rt, step)
        _, kp, vp = pools(step)
        q, k, v = step.q.to(DEV), step.k.to(DEV), step.v.to(DEV)
        eager = torch.ops.gaudirt._paged_attn_biased(q, k, v, kp, vp, md, slopes, 64, step.scale)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = torch.ops.gaudirt._paged_attn_biased(q, k, v, kp, vp, md, slopes, 64, step.scale)
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, eager)
        stream.synchronize()
    with pytest.raises(RuntimeError, match="stream"):          # a plan belongs to the stream it was built on
        torch.ops.gaudirt._paged_attn_biased(q, k, v, kp, vp, md, slopes, 64, step.scale)
