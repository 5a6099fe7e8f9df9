"""Query rows that begin anywhere: the kernels give the same bits for a packed matrix, for column slices whose rows are 4- and
2-byte aligned, and for rows whose alignment changes from one to the next."""
import pytest
import torch

from tests import steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("geometry", [(8, 2, 128), (4, 4, 64), (6, 2, 64), (16, 1, 256), (5, 1, 128)])
def test_alignment_of_query_rows_changes_no_bit(geometry):
    import gaudirt_b200 as rt
    step = steps.shared_step([300], [(0, 40, 1), (0, 7, 150), (-1, 90, 65), (0, 0, 3), (0, 100, 1)], *geometry, 16, seed=47)
    pool = step.stored_pool().to(DEV)
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    slopes = steps.slopes_of(step.q_heads).to(DEV)
    width = step.q_heads * step.head_dim

    def outputs(q):
        for share in (False, True):
            md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
            if share:
                md._share_prefixes_(step.groups, step.prefixes)
                md._set_prefix_sharing(1, 0)
            yield torch.ops.gaudirt._paged_attn_stored(q, kp, vp, md, step.head_dim, step.scale)
            yield torch.ops.gaudirt._paged_attn_biased(q, None, None, kp, vp, md, slopes, step.head_dim, step.scale)

    expected = list(outputs(step.q.to(DEV)))
    steps.check(expected[0], *steps.attend64(step, step.stored_pool()))
    for offset, pad in ((1, 8), (2, 8), (0, 1), (1, 1), (3, 7), (0, 4)):
        wide = torch.full((len(step.q), width + pad + offset), float("nan"), dtype=torch.bfloat16, device=DEV)
        q = wide[:, offset:offset + width]
        q.copy_(step.q)
        for got, want in zip(outputs(q), expected):
            assert torch.equal(got, want), (offset, pad)
    # the matrix ends where its last row ends
    tight = torch.empty(len(step.q) * width + 1, dtype=torch.bfloat16, device=DEV)[1:].view(-1, width)
    tight.copy_(step.q)
    for got, want in zip(outputs(tight), expected):
        assert torch.equal(got, want)
    assert rt._C._take_device_status() == 0
