"""Host half of the shared-prefix and two-way plans, without a GPU: every row attends to each of its keys exactly once,
every split state has one writer and one place, and what cannot be planned is refused."""
import ctypes as C
import random

import numpy as np
import pytest

from gaudirt_b200 import abi

INVALID, UNSUPPORTED, CAPACITY = 1, 2, 4


def ptr(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def build(seq, groups, prefixes, q_heads, kv_heads, head_dim, window=-1, two_way=None, split=0, pieces=0, min_saved=0, sms=148,
          shrink=0):
    lib = abi.lib()
    as32 = lambda x: None if x is None else np.ascontiguousarray(x, dtype=np.int32)  # noqa: E731
    seq, groups, prefixes, two_way = as32(seq), as32(groups), as32(prefixes), as32(two_way)
    counts = [C.c_int64() for _ in range(5)]
    refs, form = [C.byref(c) for c in counts], C.c_int()

    def call(work, combine, prefix, rows, caps):
        return lib.gk_shared_prefix_plan_build(ptr(seq), len(seq), ptr(two_way), ptr(groups), ptr(prefixes), len(prefixes),
                                               q_heads, kv_heads, head_dim, window, sms, split, pieces, min_saved, C.byref(form), ptr(work),
                                               caps[0], refs[0], ptr(combine), caps[1], refs[1], refs[2], ptr(prefix), caps[3],
                                               refs[3], ptr(rows), caps[4], refs[4])

    rc = call(None, None, None, None, [0] * 5)
    if rc:
        return rc
    n = [c.value for c in counts]
    arrays = [np.zeros((max(1, k), w), dtype=np.int32) for k, w in zip((n[0], n[1], n[3], n[4]), (8, 4, 8, 4))]
    rc = call(*arrays, [n[0], n[1], n[2], n[3], n[4] - shrink])
    if rc:
        return rc
    assert [c.value for c in counts] == n
    work, combine, prefix, rows = (a[:k] for a, k in zip(arrays, (n[0], n[1], n[3], n[4])))
    assert not form.value & 1 or all(w[1] <= 128 // (q_heads // kv_heads) for w in prefix)
    return work, combine, n[2], prefix, rows


def check_cover(seq, plan, q_heads, kv_heads, window, two_way):
    work, combine, entries, prefix, rows = plan
    where, seen, states = {}, {}, {}
    for s, (first, n, pos, table_row) in enumerate(seq):
        for r in range(n):
            p = pos + r
            low = max(0, p - window + 1) if window > 0 else 0
            where[first + r] = (p, low, max(p, (two_way[s] if two_way else 0) - 1), table_row)
            seen[first + r] = []
    for first, n, pos, table_row, lo, hi, base, parts in work.tolist():
        for r in range(n):
            assert where[first + r][0] == pos + r and where[first + r][3] == table_row
            seen[first + r].append((lo, hi))
            if base >= 0:
                for h in range(q_heads):
                    entry = base + r * q_heads + h
                    assert entry not in states and 0 <= entry < entries
                    states[entry] = (first + r, h, parts >> 16)
            else:
                assert parts & 0xffff == 1
    for at, n, part, table_row, lo, hi, highest, zero in prefix.tolist():
        assert zero == 0 and 0 < n <= 2 * (128 // (q_heads // kv_heads)) and lo < hi
        assert highest == max(rows[at + i][1] for i in range(n))
        for row, p, entry0, stride in rows[at:at + n].tolist():
            assert where[row][0] == p and hi <= p
            seen[row].append((lo, hi))
            for h in range(q_heads):
                entry = entry0 + part * stride + h
                assert entry not in states and 0 <= entry < entries
                states[entry] = (row, h, part)
    assert len(states) == entries
    for row, ranges in seen.items():
        p, low, last, _ = where[row]
        keys = sorted((max(lo, low), hi) for lo, hi in ranges if hi > low)      # a window hides the keys below `low`
        assert keys[-1][1] == max(hi for _, hi in keys) > last
        assert keys[0][0] == low
        assert all(a[1] == b[0] for a, b in zip(keys, keys[1:])), (row, keys)
    for first, n, base, parts in combine.tolist():                 # the states of a block stand in part order
        for part in range(parts):
            for r in range(n):
                for h in range(q_heads):
                    assert states[base + (part * n + r) * q_heads + h] == (first + r, h, part)


@pytest.mark.parametrize("seed", range(40))
def test_every_key_once(seed):
    rng = random.Random(seed)
    q_heads, kv_heads = rng.choice([(8, 2), (4, 4), (16, 1), (6, 2), (5, 1)])
    head_dim = rng.choice([64, 128, 256])
    prefixes = [rng.choice([0, 1, 63, 64, 128, 500, 3000]) for _ in range(rng.randint(1, 4))]
    seq, groups, two_way, row = [], [], [], 0
    for s in range(rng.randint(1, 30)):
        g = rng.randint(-1, len(prefixes) - 1)
        n, pos = rng.choice([1, 1, 1, 2, 5, 20]), (prefixes[g] if g >= 0 else 0) + rng.choice([0, 1, 40, 700])
        seq.append((row, n, pos, s))
        groups.append(g)
        two_way.append(rng.choice([0, 0, pos, pos + n]))
        row += n
    window = rng.choice([-1, -1, 1, 50, 600])
    two_way = two_way if rng.random() < 0.5 else None
    plan = build(seq, groups, prefixes, q_heads, kv_heads, head_dim, window, two_way, rng.choice([0, 64, 256]),
                 rng.choice([0, 64, 128, 1000]), sms=rng.choice([1, 8, 148]))
    check_cover(seq, plan, q_heads, kv_heads, window, two_way)


def test_without_groups_the_plan_is_the_ordinary_one():
    lib = abi.lib()
    seq = np.array([(0, 1, 5000, 0), (1, 3, 700, 1), (4, 1, 0, 2)], dtype=np.int32)
    counts = [C.c_int64() for _ in range(3)]
    work, combine = np.zeros((400, 8), dtype=np.int32), np.zeros((400, 4), dtype=np.int32)
    assert lib.gk_attention_plan_build(ptr(seq), 3, 8, 2, 128, -1, 148, 0, ptr(work), 400, C.byref(counts[0]), ptr(combine), 400,
                                       C.byref(counts[1]), C.byref(counts[2])) == 0
    plan = build(seq, [-1, -1, -1], [], 8, 2, 128)
    assert np.array_equal(plan[0], work[:counts[0].value]) and np.array_equal(plan[1], combine[:counts[1].value])
    assert plan[2] == counts[2].value and len(plan[3]) == 0 and len(plan[4]) == 0


def test_a_prefix_is_read_together_where_that_saves_enough():
    seq = [(i, 1, 1000 + i, i) for i in range(4)]
    saved = 3 * 1000 * 2 * 128 * 4
    for least, shared in ((saved, True), (saved + 1, False)):
        plan = build(seq, [0] * 4, [1000], 8, 2, 128, min_saved=least)
        assert (len(plan[3]) > 0) == shared
    assert len(build(seq, [0, -1, -1, -1], [1000], 8, 2, 128)[3]) == 0          # nobody to share with
    assert len(build(seq, [0] * 4, [1000], 8, 2, 128, window=1)[3]) == 0         # nobody sees the prefix


def test_refusals():
    seq = [(0, 1, 100, 0), (1, 2, 90, 1)]
    assert build(seq, [0, 0], [91], 8, 2, 128) == INVALID           # a row inside the prefix
    assert build(seq, [0, 1], [90], 8, 2, 128) == INVALID           # no such group
    assert build(seq, [0, -2], [90], 8, 2, 128) == INVALID
    assert build(seq, [0, 0], [-1], 8, 2, 128) == INVALID
    assert build(seq, [0, 0], [90], 8, 2, 128, two_way=[0, 93]) == INVALID       # past the last row
    assert build(seq, [0, 0], [90], 8, 2, 128, two_way=[-1, 0]) == INVALID
    assert build(seq, [0, 0], [90], 8, 2, 128, window=0) == INVALID
    assert build(seq, [0, 0], [90], 8, 3, 128) == UNSUPPORTED
    assert build(seq, [0, 0], [90], 8, 2, 96) == UNSUPPORTED
    assert build(seq, [0, 0], [90], 34, 2, 128) == UNSUPPORTED
    assert build(seq, [0, 0], [90], 8, 2, 128, shrink=1) == CAPACITY
    assert build([(0, 1, 2**31 - 1, 0), (1, 1, 5, 1)], [0, 0], [5], 8, 2, 128) == INVALID
    # lists that cannot be held end as an error code, not as an exception through a C entry
    lib, sizes = abi.lib(), [C.byref(C.c_int64()) for _ in range(5)]
    one = np.array(seq, dtype=np.int32)
    assert lib.gk_shared_prefix_plan_build(ptr(one), 2, None, ptr(one), ptr(one), 2**60, 8, 2, 128, -1, 148, 0, 0, 0, C.byref(C.c_int()),
                                           None, 0, sizes[0], None, 0, sizes[1], sizes[2], None, 0, sizes[3], None, 0, sizes[4]) == CAPACITY


def test_two_way_prefill_records():
    lib = abi.lib()
    seq = np.array([(0, 300, 50, 0), (300, 1, 9, 1), (301, 40, 0, 2)], dtype=np.int32)
    two_way = np.array([350, 10, 7], dtype=np.int32)
    n, rest = C.c_int64(), C.c_int64()
    work, left = np.zeros((64, 8), dtype=np.int32), np.zeros((3, 4), dtype=np.int32)
    assert lib.gk_prefill_plan_build_two_way(ptr(seq), 3, ptr(two_way), 8, 2, -1, 0, ptr(work), 64, C.byref(n), ptr(left),
                                             C.byref(rest)) == 0
    assert rest.value == 1 and left[0].tolist() == [300, 1, 9, 1]
    for first, rows, pos, table_row, lo, hi, *_ in work[:n.value].tolist():
        assert lo == 0 and hi == max(pos + rows, int(two_way[table_row]))
    two_way[0] = 351
    assert lib.gk_prefill_plan_build_two_way(ptr(seq), 3, ptr(two_way), 8, 2, -1, 0, ptr(work), 64, C.byref(n), ptr(left),
                                             C.byref(rest)) == INVALID


def test_launch_arguments_are_judged_on_the_host():
    """Refused before anything is launched (there is no GPU here)."""
    lib = abi.lib()
    one = C.c_void_p(4096)
    extend = [one, 4, 16, 16, one, one, one, 3, one, 5, one, 16, 8, None, one, one, one, one, one, one, None, None]
    for at, value in ((0, None), (4, None), (7, 0), (8, None), (3, 15), (11, 0), (12, 0), (2, 0), (2, 2**31), (9, -1), (7, 4097)):
        args = list(extend)
        args[at] = value
        assert lib.gk_extend_requests(*args) == INVALID, at
    assert lib.gk_extend_requests(*[*extend[:7], 65537, *extend[8:13], one, *extend[14:]]) == UNSUPPORTED
    assert lib.gk_extend_requests(one, 262145, *extend[2:]) == UNSUPPORTED
    size = C.c_uint64()
    assert lib.gk_extend_requests_workspace_bytes(4096, C.byref(size)) == 0 and size.value == 0
    assert lib.gk_extend_requests_workspace_bytes(4097, C.byref(size)) == 0 and size.value == 4097 * 8 + 24
    assert lib.gk_extend_requests_workspace_bytes(0, C.byref(size)) == INVALID
    check = [one, 4, 16, 16, None, 4, one, 2, one, None, None]
    for at, value in ((0, None), (6, None), (8, None), (3, 15), (5, 0), (6, C.c_void_p(4100)), (7, -1)):
        args = list(check)
        args[at] = value
        assert lib.gk_shared_prefix_check(*args) == INVALID, at
    attend = [one, 1024, one, one, 64, one, 16, 1, 1, None, one, 1, 0, one, one, one, None, 1.0, 0.0, -1, 8, 2, 128, None, None]
    for at, value in ((0, None), (10, None), (13, None), (14, None), (15, None), (13, C.c_void_p(4100)), (16, C.c_void_p(4097)),
                      (17, 0.0), (18, -1.0), (19, 0), (8, 3)):
        args = list(attend)
        args[at] = value
        assert lib.gk_shared_prefix_attn_bf16(*args) == INVALID, at
    for at, value in ((20, 34), (22, 96)):
        args = list(attend)
        args[at] = value
        assert lib.gk_shared_prefix_attn_bf16(*args) == UNSUPPORTED, at
    extended = [one, 1024, None, None, 0, 0, None, one, one, 64, one, 16, 1, 1, None, one, 1, one, 1, (C.c_void_p * 1)(4096), 1, 1024,
                one, one, None, None, None, 4, 1.0, 0.0, -1, 8, 2, 128, None, None]
    for at, value in ((0, None), (15, None), (17, None), (18, -1), (16, 0), (22, None), (24, one), (25, C.c_void_p(4097)),
                      (26, C.c_void_p(4098)), (27, 8), (28, 0.0), (2, one)):
        args = list(extended)
        args[at] = value
        assert lib.gk_paged_attn_extended_multi_bf16(*args) == INVALID, at
    for at, value in ((31, 34), (33, 96)):
        args = list(extended)
        args[at] = value
        assert lib.gk_paged_attn_extended_multi_bf16(*args) == UNSUPPORTED, at
    args = list(extended)
    args[16] = args[18] = 0                                        # nothing to do is not an error
    assert lib.gk_paged_attn_extended_multi_bf16(*args) == 0
