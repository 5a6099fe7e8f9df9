"""The status word reports what was only launched; a call that raises its own error adds nothing to it and takes nothing out."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BAD_METADATA = 8


def refused_metadata(rt):
    """Two rows that name one slot."""
    table = torch.arange(32, dtype=torch.int32, device=DEV).view(2, 16).contiguous()
    batch = torch.arange(2, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="invalid scheduler metadata"):
        rt.PagedMetadata.from_device(torch.tensor([3, 3], dtype=torch.int32, device=DEV), batch,
                                     torch.tensor([3, 3], dtype=torch.int32, device=DEV), table, [3, 3], [1, 1], 32)


def refused_batch(rt):
    """A request that the table does not have: nothing but the status word says so."""
    one = torch.zeros(1, dtype=torch.int64, device=DEV)
    rt._C._extend_paged_requests(torch.full((2, 32), -1, dtype=torch.int32, device=DEV),
                                 torch.tensor([5], dtype=torch.int32, device=DEV), one, torch.ones_like(one).int(), one, one, 16, 1)


def test_refused_metadata_leaves_the_word_alone():
    import gaudirt_b200 as rt
    rt._C._take_device_status()
    refused_metadata(rt)
    assert rt._C._take_device_status() == 0
    refused_batch(rt)
    refused_metadata(rt)
    assert rt._C._take_device_status() == BAD_METADATA
    refused_metadata(rt)
    assert rt._C._take_device_status() == 0
