"""Slots that no row of the step sees are never looked at: uninitialised ends of pages, pages of other sequences, and cached
tokens in front of every row's window may hold anything, NaN and infinities included."""
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


def poisoned(step, window, value):
    """The step's pool with `value` in every slot that no row sees."""
    seen = torch.zeros(step.slots, dtype=torch.bool)
    for i, (c, n) in enumerate(zip(step.cached, step.lengths)):
        first = max(0, c - window + 1) if window > 0 else 0
        seen[step.mapping[i, first:c + n].long()] = True
    pool = step.stored_pool()
    pool[:, :, ~seen] = value
    assert (~seen).any()
    return pool.to(DEV)


SHARED = ([400, 37], [(0, 100, 1), (0, 0, 1), (1, 20, 3), (0, 250, 1), (-1, 130, 2), (1, 5, 1), (0, 60, 90), (-1, 3, 40)])


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("window", [-1, 60, 150, 333])
@pytest.mark.parametrize("page", [1, 16, 128])
@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 4, 64), (16, 1, 256)])
def test_unseen_slots(rt, geometry, page, window, value):
    step = steps.shared_step(*SHARED, *geometry, page, seed=53)
    pool = poisoned(step, window, value)
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    q, slopes = step.q.to(DEV), steps.slopes_of(step.q_heads)
    for share in (False, True):
        for bias in (None, slopes):
            md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
            if share:
                md._share_prefixes_(step.groups, step.prefixes)
                md._set_prefix_sharing(1, 0)
            if bias is None:
                out = torch.ops.gaudirt._paged_attn_stored(q, kp, vp, md, step.head_dim, step.scale, 0.0, window)
            else:
                out = torch.ops.gaudirt._paged_attn_biased(q, None, None, kp, vp, md, bias.to(DEV), step.head_dim, step.scale,
                                                           0.0, window)
            steps.check(out, *steps.attend64(step, step.stored_pool(), 0.0, window, bias))
    assert rt._C._take_device_status() == 0


@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("window", [-1, 200])
def test_unseen_slots_in_every_staging(rt, form, window):
    """Short tails of two warps included."""
    step = steps.shared_step([256], [(0, (i * 37) % 200, 1) for i in range(130)], 32, 8, 128, 32, seed=31)
    pool = poisoned(step, window, float("nan"))
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    assert rt.abi.lib().gk_set_attention_form(form) == 0
    try:
        for share in (False, True):
            md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
            if share:
                md._share_prefixes_(step.groups, step.prefixes)
                md._set_prefix_sharing(1, 0)
            out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, 128, step.scale, 0.0, window)
            steps.check(out, *steps.attend64(step, step.stored_pool(), 0.0, window))
    finally:
        rt.abi.lib().gk_set_attention_form(0)


@pytest.mark.parametrize("min_rows", [0, -1])
@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 4, 64), (16, 1, 256)])
def test_unseen_slots_behind_two_way_prefixes(rt, geometry, min_rows):
    step = steps.plain_step([100, 90, 300, 0], [260, 37, 4, 5], *geometry, 128, seed=59, two_way=[359, 100, 302, 5])
    md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
    md._set_prefix_mask_(step.two_way)
    md._set_prefill_min_rows(min_rows)
    pool = poisoned(step, -1, float("nan"))
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), kp, vp, md, step.head_dim, step.scale)
    steps.check(out, *steps.attend64(step, step.stored_pool()))


@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 4, 64), (16, 1, 256)])
def test_entries_that_a_scheduler_took_back(rt, geometry):
    """A scheduler that frees the pages in front of the window leaves no slot in their table cells."""
    window = 150
    step = steps.shared_step([400], [(0, 100, 1), (0, 0, 1), (0, 20, 3), (0, 140, 1)], *geometry, 16, seed=61)
    table = step.mapping.clone()
    lowest = min(step.cached) - window + 1
    for i, c in enumerate(step.cached):
        table[i, :lowest] = -1                                 # nobody sees these
    pool = step.stored_pool().to(DEV)
    batch = torch.arange(len(step.cached), dtype=torch.int32, device=DEV)
    for share in (False, True):
        md = rt.PagedMetadata._from_scheduler(step.locations.to(DEV), batch, step.positions.to(torch.int32).to(DEV),
                                              table.to(DEV), step.cached, step.lengths, step.slots, None, 0)
        if share:
            md._share_prefixes_(step.groups, step.prefixes)
            md._set_prefix_sharing(1, 0)
        out = torch.ops.gaudirt._paged_attn_stored(step.q.to(DEV), pool[0].transpose(0, 1), pool[1].transpose(0, 1), md,
                                                   step.head_dim, step.scale, 0.0, window)
        steps.check(out, *steps.attend64(step, step.stored_pool(), 0.0, window))
        assert rt._C._take_device_status() == 0
