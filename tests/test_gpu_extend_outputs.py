"""The six outputs of the slot-map operator are tensors of their own: aligned, in storages of their own, as the operator's
schema and its shape function say."""
import io

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def arguments(batch, page=16):
    """Empty requests that append one token each."""
    return (torch.full((batch, page), -1, dtype=torch.int32, device=DEV), torch.arange(batch, dtype=torch.int32, device=DEV),
            torch.zeros(batch, dtype=torch.int64, device=DEV), torch.ones(batch, dtype=torch.int32, device=DEV),
            torch.arange(batch, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV), page, batch + 3)


@pytest.mark.parametrize("batch", [1, 2, 3, 4, 33, 4097])
def test_outputs_are_tensors_of_their_own(batch):
    import gaudirt_b200 as rt
    args = arguments(batch)
    out = rt._C._extend_paged_requests(*args)
    fake = torch._subclasses.FakeTensorMode()
    with fake:
        shapes = torch.ops.gaudirt._extend_paged_requests(*(fake.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args))
    for got, want in zip(out, shapes):
        assert got.dtype == want.dtype and got.shape == want.shape and got.stride() == want.stride()
        assert got.storage_offset() == want.storage_offset() == 0
        assert got.data_ptr() % 16 == 0
        assert got.untyped_storage().nbytes() == got.numel() * got.element_size()
    assert len({t.untyped_storage().data_ptr() for t in out}) == 6
    buffer = io.BytesIO()
    torch.save(out, buffer)
    buffer.seek(0)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(out, torch.load(buffer)))


@pytest.mark.parametrize("batch", [1, 5])
def test_schema_and_shapes(batch):
    import gaudirt_b200  # noqa: F401
    torch.library.opcheck(torch.ops.gaudirt._extend_paged_requests.default, arguments(batch),
                          test_utils=("test_schema", "test_faketensor"))
