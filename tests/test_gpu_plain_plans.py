"""Plans of steps that declare nothing: the records of the ordinary builders, whatever the mix of rows."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def metadata(rt, cached, new, page=16):
    context = -(-max(c + n for c, n in zip(cached, new)) // page) * page
    table = torch.arange(len(cached) * context, dtype=torch.int32).view(-1, context)
    requests = torch.arange(len(cached)).repeat_interleave(torch.tensor(new))
    positions = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)])
    return rt.PagedMetadata(table[requests, positions].contiguous(), requests, positions, table, table.numel())


def ordinary(lib, md, q_heads, kv_heads, head_dim, window, min_rows):
    """Words of the plan from the C entries: decode records, combine records, prefill records."""
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    seq = np.array(md.sequences(), dtype=np.int32).reshape(-1, 4)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n_tc, n_left = C.c_int64(0), C.c_int64(len(seq))
    left, tc = seq.copy(), np.zeros((4096, 8), dtype=np.int32)
    if min_rows >= 0:
        assert lib.gk_prefill_plan_build(ptr(seq), len(seq), q_heads, kv_heads, window, min_rows, ptr(tc), 4096, C.byref(n_tc),
                                         ptr(left), C.byref(n_left)) == 0
    work, combine = np.zeros((8192, 8), dtype=np.int32), np.zeros((8192, 4), dtype=np.int32)
    n_work, n_combine, entries = C.c_int64(0), C.c_int64(0), C.c_int64(0)
    if n_left.value:
        assert lib.gk_attention_plan_build(ptr(left), n_left.value, q_heads, kv_heads, head_dim, window, sms, 0, ptr(work), 8192,
                                           C.byref(n_work), ptr(combine), 8192, C.byref(n_combine), C.byref(entries)) == 0
    return np.concatenate([work[:n_work.value].reshape(-1), combine[:n_combine.value].reshape(-1), tc[:n_tc.value].reshape(-1)])


@pytest.mark.parametrize("min_rows", [0, -1, 1, 40])
@pytest.mark.parametrize("window", [-1, 300])
@pytest.mark.parametrize("cached,new", [([700], [1]), ([0, 90, 1000, 5], [40, 1, 130, 3]), ([100] * 70, [1] * 70),
                                        ([3000, 10, 2000], [1, 300, 2]), ([0, 0], [64, 200])])
def test_records_are_the_ordinary_ones(cached, new, window, min_rows):
    import gaudirt_b200 as rt
    lib = rt.abi.lib()
    for declare in ("nothing", "no_group", "causal", "sharing_off"):
        md = metadata(rt, cached, new)
        md._set_prefill_min_rows(min_rows)
        if declare == "no_group":
            md._share_prefixes_([-1] * len(cached), [])
        elif declare == "causal":
            md._set_prefix_mask_([0] * len(cached))
        elif declare == "sharing_off":
            md._share_prefixes_([0] + [-1] * (len(cached) - 1), [cached[0]])
            md._set_prefix_sharing(0, 0)
        plan = md.attention_plan_for(8, 2, 128, window).cpu().numpy()
        want = ordinary(lib, md, 8, 2, 128, window, min_rows)
        assert np.array_equal(plan[:len(want)], want) and len(plan) == max(4, len(want)), declare
