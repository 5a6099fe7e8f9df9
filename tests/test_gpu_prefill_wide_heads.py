"""head_dim 256 of the tensor-core prefill kernel: scores run two KV tiles ahead of the products with V, so the last product
must be waited for by itself.  Ranges of exactly two, three and a few KV tiles, keys and values cold in L2, the same bits on
every launch."""
import pytest
import torch

from tests.test_gpu_prefill import run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [128, 1])
@pytest.mark.parametrize("prefix", [50, 100, 150, 230])
def test_ranges_of_a_few_tiles(prefix, page):
    """64-token tiles: prefixes of 50, 100, 150 and 230 and 20 new rows make 2, 2, 3 and 4 of them."""
    n_tc, n_rest = run_case([(prefix, 20)] * 40, 8, 2, page, seed=prefix + page, d=256)
    assert n_tc == 40 and n_rest == 0


def test_same_bits_on_every_launch():
    import gaudirt_b200 as rt
    n, prefix, new, d, heads = 48, 90, 30, 256, 8
    slots = n * 128
    mapping = torch.arange(slots, dtype=torch.int32).view(n, 128)
    requests = torch.arange(n).repeat_interleave(new)
    positions = torch.arange(prefix, prefix + new).repeat(n)
    md = rt.PagedMetadata(mapping[requests, positions].contiguous(), requests, positions, mapping, slots)
    gen = torch.Generator(device="cuda").manual_seed(1)
    pool = torch.randn(2, 2, slots, d, generator=gen, device="cuda").to(torch.bfloat16)
    q = torch.randn(n * new, heads * d, generator=gen, device="cuda").to(torch.bfloat16)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    first = None
    for _ in range(8):
        flush.zero_()
        out = torch.ops.gaudirt._paged_attn_stored(q, pool[0].transpose(0, 1), pool[1].transpose(0, 1), md, d, d ** -0.5)
        first = out if first is None else first
        assert torch.equal(out, first)
