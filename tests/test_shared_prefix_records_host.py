"""Where the records of a shared prefix begin: at the first key that any row of the group sees, and behind that at whole tiles
of the kernel."""
import random

import pytest

from tests.test_operator_plans_host import build


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("seed", range(8))
def test_records_begin_where_the_windows_do(head_dim, seed):
    rng = random.Random(seed)
    tile = 64 if head_dim == 256 else 128
    window = rng.choice([-1, 60, 200, 777, 3000])
    prefixes = [rng.choice([1, 100, 640, 3000]) for _ in range(3)]
    seq, groups, row = [], [], 0
    for s in range(20):
        g = rng.randrange(3)
        n = rng.choice([1, 1, 2, 4])
        seq.append((row, n, prefixes[g] + rng.choice([0, 1, 40, 300]), s))
        groups.append(g)
        row += n
    plan = build(seq, groups, prefixes, 8, 2, head_dim, window, pieces=rng.choice([0, 128, 512]))
    work, combine, entries, prefix, rows = plan
    group_of = {first + r: g for (first, n, _, _), g in zip(seq, groups) for r in range(n)}
    for g in range(3):
        members = [s for s, other in zip(seq, groups) if other == g]
        low = min(max(0, pos - window + 1) if window > 0 else 0 for _, _, pos, _ in members)
        records = [w for w in prefix.tolist() if group_of[int(rows[w[0]][0])] == g]
        assert bool(records) == (len(members) > 1 and low < prefixes[g])
        for first, n, part, table_row, begin, end, highest, zero in records:
            assert begin == low if part == 0 else begin % tile == 0 and begin > low
            assert end == prefixes[g] or end % tile == 0
