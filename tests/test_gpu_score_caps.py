"""Caps of any size in the kernels that carry a distance bias, a two-way prefix or a shared prefix: loose caps leave ordinary
scores alone, and one huge score does not cost its neighbours their digits."""
import pytest
import torch

from tests import steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GEOMETRIES = [(8, 2, 128), (4, 4, 64), (16, 1, 256)]


@pytest.fixture(scope="module")
def rt():
    import gaudirt_b200
    gaudirt_b200._C._take_device_status()
    return gaudirt_b200


def outputs(rt, step, softcap, window=-1):
    """The step through the shared-prefix kernels and through the biased ones, each with its slopes (None, then one per head)."""
    pool = step.stored_pool().to(DEV)
    kp, vp = pool[0].transpose(0, 1), pool[1].transpose(0, 1)
    q, slopes = step.q.to(DEV), steps.slopes_of(step.q_heads)
    for share in (True, False):
        md = rt.PagedMetadata(step.locations, step.requests, step.positions, step.mapping, step.slots)
        if share:
            md._share_prefixes_(step.groups, step.prefixes)
            md._set_prefix_sharing(1, 0)
            yield None, torch.ops.gaudirt._paged_attn_stored(q, kp, vp, md, step.head_dim, step.scale, softcap, window)
            assert md._last_plan_prefix_records() > 0
        yield slopes, torch.ops.gaudirt._paged_attn_biased(q, None, None, kp, vp, md, slopes.to(DEV), step.head_dim, step.scale,
                                                           softcap, window)


MEMBERS = [(0, 40, 1), (0, 0, 3), (-1, 90, 1), (0, 100, 1), (0, 7, 150)]


# A loose cap leaves a score of ordinary size what it is to 2^-20 of itself: with |scores| below 16 an error of 2^-16, an
# eighth of a probability's half step in bf16 being 2^-11, so the bound of `steps.check` covers it.
@pytest.mark.parametrize("softcap", [1e3, 1e4, 1e5, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_loose_caps(rt, geometry, softcap):
    step = steps.shared_step([300], MEMBERS, *geometry, 16, seed=29)
    for slopes, out in outputs(rt, step, softcap):
        steps.check(out, *steps.attend64(step, step.stored_pool(), softcap, slopes=slopes))


def huge_score_range(step, softcap, at, slopes):
    """(lowest, highest, weighted |v|) of every output in binary64 when the raw scores of the keys at positions `at` are only
    known to the rounding of their sum: d products added in fp32 one after another are off by at most d * 2^-23 of the sum of
    their sizes (2^-23, not 2^-24, for sums that truncate), which is nothing next to a score of ordinary size but 10 to 100
    where huge products cancel.  An output is a ratio of two functions linear in each key's exponential, so it is monotone in
    each such score and its extremes are at the corners."""
    pool, d, share = step.stored_pool(), step.head_dim, step.q_heads // step.kv_heads
    lowest, highest, sizes, first = [], [], [], 0
    for c, n in zip(step.cached, step.lengths):
        end = c + n
        slots = step.mapping[len(lowest), :end].long()
        k, v = (pool[x][:, slots].double().repeat_interleave(share, 0) for x in (0, 1))
        q = step.q[first:first + n].double().view(n, step.q_heads, d).transpose(0, 1)
        raw, off = (q @ k.transpose(1, 2)) * step.scale, (q.abs() @ k.abs().transpose(1, 2)) * (step.scale * d * 2.0 ** -23)
        p, j = torch.arange(c, end)[:, None], torch.arange(end)[None, :]
        inside = [x for x in at if x < end]
        outs, size = [], None
        for corner in range(2 ** len(inside)):
            s = raw.clone()
            for bit, x in enumerate(inside):
                s[..., x] += off[..., x] if corner >> bit & 1 else -off[..., x]
            s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes.double()[:, None, None] * (p - j).abs()
            w = torch.softmax(s.masked_fill(j > p, float("-inf")), -1)
            outs.append((w @ v).transpose(0, 1).reshape(n, -1))
            each = (w @ v.abs()).transpose(0, 1).reshape(n, -1)
            size = each if size is None else torch.maximum(size, each)
        lowest.append(torch.stack(outs).amin(0))
        highest.append(torch.stack(outs).amax(0))
        sizes.append(size)
        first += n
    return torch.cat(lowest), torch.cat(highest), torch.cat(sizes)


# Every sequence has one key (two: one in the prefix, one behind it) whose scores are as large as the cap.  A row either
# gives it everything or nothing; what it leaves is judged by the scores of ordinary size next to it, as above.
@pytest.mark.parametrize("softcap", [1e4, 1e6])
@pytest.mark.parametrize("at", [(17,), (290, 20)])
@pytest.mark.parametrize("geometry", GEOMETRIES)
def test_one_huge_score_among_ordinary_ones(rt, geometry, at, softcap):
    step = steps.shared_step([300], MEMBERS, *geometry, 16, seed=31)
    for position in at:
        slots = torch.unique(step.mapping[:, position])
        slots = slots[slots >= 0].long()
        step.pool[0][:, slots] = (step.pool[0][:, slots].float() * softcap).to(torch.bfloat16)
    for slopes, out in outputs(rt, step, softcap):
        low, high, size = huge_score_range(step, softcap, at, slopes)
        got = out.cpu().double()
        assert ((high - low).amax(-1) < 1e-3).double().mean() > 0.9           # nearly every row is known to the last digit
        steps.check(out, torch.minimum(torch.maximum(got, low), high), size)
