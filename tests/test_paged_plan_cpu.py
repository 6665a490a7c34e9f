"""kata_paged_decode_plan with tiles of 64 slots (int8 heads of 128) beside 16 and 32, and where the cuts of long lists fall: no piece of a few tiles, no share above the others."""
import bisect
import random

import pytest

from .test_paged_cpu import L, _plan  # noqa: F401

PAD, SNAP = 8, 4   # a segment counts as 8 tiles more, and a cut within 4 tiles of its end moves there, once a CTA's share is 32 tiles or more


def _check(L, keys, kvh, tile, sm=148):  # noqa: F811
    c, first, most = _plan(L, keys, kvh, tile, sm)
    nt = [max(1, -(-k // tile)) for k in keys for _ in range(kvh)]
    total = sum(nt)
    assert 1 <= c <= sm and first[0] == 0 and first[-1] == total and all(a <= b for a, b in zip(first, first[1:])), (keys, kvh, tile)
    worst, start, equal = 0, 0, len(set(nt)) == 1
    cuts = sorted(set(first))
    for t in nt:
        inside = bisect.bisect_left(cuts, start + t) - bisect.bisect_right(cuts, start)
        worst = max(worst, inside + 1)
        if total >= sm * 4 * PAD and not equal:
            for x in cuts[bisect.bisect_right(cuts, start):bisect.bisect_left(cuts, start + t)]:
                assert SNAP < x - start < t - SNAP, (keys, kvh, tile, x - start, t)   # no piece of 1 to 4 tiles at either end
        start += t
    assert worst == most
    if not equal:   # a share of the list with its pads, a cut moved at either end, and the rounding
        pad = PAD if total >= sm * 4 * PAD else 0
        assert max(b - a for a, b in zip(first, first[1:])) <= (total + len(nt) * pad) / c + 2 * SNAP + 1


@pytest.mark.parametrize("keys,kvh", [([15000] * 18, 8), ([1000, 20000, 7, 0, 13000, 64, 65, 4096], 8), ([524288] * 3, 16), ([0] * 256, 16), ([63], 1), ([32768], 8), ([1 + 77 * i for i in range(256)], 3)])
def test_tiles_of_64_slots(L, keys, kvh):  # noqa: F811
    _check(L, keys, kvh, 64)


def test_random_batches(L):  # noqa: F811
    rng = random.Random(12)
    for _ in range(400):
        top = rng.choice([1, 200, 5000, 33000])
        keys = [rng.randint(0, top) for _ in range(rng.randint(1, 256))] if rng.random() < 0.8 else [rng.randint(0, top)] * rng.randint(1, 60)
        _check(L, keys, rng.randint(1, 16), rng.choice([16, 32, 64]), rng.choice([148, 148, 132, 16, 1]))
