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


def test_a_step_that_needs_no_page_takes_an_empty_free_list():
    import gaudirt_b200 as rt
    table = torch.full((3, 64), -1, dtype=torch.int32, device=DEV)
    table[2, :5] = torch.arange(32, 37, dtype=torch.int32, device=DEV)
    out = rt._C._extend_paged_requests(table, torch.tensor([2], dtype=torch.int32, device=DEV), torch.tensor([5], device=DEV),
                                       torch.tensor([11], dtype=torch.int32, device=DEV),
                                       torch.empty(0, dtype=torch.int64, device=DEV), torch.tensor([0], device=DEV), 16, 11)
    assert out[0].tolist() == list(range(37, 48)) and out[1].tolist() == list(range(5, 16)) and int(out[5]) == 0
    assert table[2].tolist() == list(range(32, 48)) + [-1] * 48 and (table[:2] == -1).all()
    assert rt._C._take_device_status() == 0


@pytest.mark.parametrize("batch", [64, 4097])
def test_two_graphs_and_an_eager_call_between_them(batch):
    """Each capture has outputs and scan room of its own: replays in turn and an eager call on another stream agree."""
    import gaudirt_b200 as rt
    expected = [t.cpu() for t in rt._C._extend_paged_requests(*arguments(batch))]
    inputs, graphs, outs = [arguments(batch) for _ in range(2)], [], []
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for args in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(rt._C._extend_paged_requests(*args))
        graphs.append(graph)
    for _ in range(3):
        for graph, args in zip(graphs, inputs):
            args[0].fill_(-1)
            graph.replay()
        with torch.cuda.stream(other):
            eager = rt._C._extend_paged_requests(*arguments(batch))
            other.synchronize()
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(out, expected))
        for args in inputs:
            assert torch.equal(args[0][:, 0].cpu(), expected[0][:batch]) and (args[0][:, 1:] == -1).all()
    assert rt._C._take_device_status() == 0
