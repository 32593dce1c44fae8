"""How the paged attention kernels cut their work, restated: every stream and block is covered once, by consecutive CTAs, and
the merge kernels find exactly the parts that were written."""
import random

import pytest


def few_cuts(streams, units, ctas, most):
    """csrc/paged_few.cu: the cuts after moving, and the records for the merge kernel {stream: (first CTA, parts)}."""
    raw = [i * units // ctas for i in range(ctas + 1)]
    where = lambda u: next(k for k, (a, b) in enumerate(streams) if a <= u < b)  # noqa: E731

    def moved(cut, s0, s1):
        return s0 if cut - s0 <= most else (s1 if s1 - cut <= most else cut)

    cuts = [moved(raw[i], *streams[where(raw[i])]) for i in range(ctas)] + [units]
    records = {}
    for i in range(ctas - 1):
        k = where(raw[i + 1])
        s0, s1 = streams[k]
        if s0 < cuts[i + 1] < s1 and raw[i] - s0 <= most:
            last = next(j for j in range(ctas) if raw[j] <= s1 - 1 < raw[j + 1])
            if last > i + 1 and s1 - raw[last] <= most:
                last -= 1
            assert k not in records
            records[k] = (i, last - i + 1)
    return cuts, records


@pytest.mark.parametrize("seed", range(8))
def test_slices_of_streams(seed):
    rng = random.Random(seed)
    for _ in range(150):
        n, hkv, hd = rng.randint(1, 40), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        streams, units = [], 0
        for length in (rng.choice([0, 1, 2, 3, rng.randint(1, 400)]) for _ in range(n)):
            for _ in range(hkv if length else 0):
                streams.append((units, units + length))
                units += length
        if not units:
            continue
        ctas = min(rng.choice([148, 296]), (units + 3) // 4)
        cuts, records = few_cuts(streams, units, ctas, min(65536 // (16 * 4 * hd), units // ctas // 2))
        assert cuts == sorted(cuts)
        begun = set()
        for k, (s0, s1) in enumerate(streams):
            owners = [i for i in range(ctas) if max(cuts[i], s0) < min(cuts[i + 1], s1)]
            if len(owners) == 1:
                assert k not in records
                continue
            assert records[k] == (owners[0], len(owners)) and owners == list(range(owners[0], owners[-1] + 1))
            assert owners[0] not in begun  # a CTA has room for one stream that begins and goes on
            begun.add(owners[0])


ITEM = 4


def tile_at(x, start, unit, nt, most):
    """csrc/paged_chunk.cu"""
    start += ITEM
    end = start + nt * unit
    if x >= end:
        return nt
    if x <= start + most:
        return 0
    return nt if x >= end - most else -(-(x - start) // unit)


@pytest.mark.parametrize("seed", range(8))
def test_slices_of_blocks(seed):
    rng = random.Random(seed)
    for _ in range(300):
        blocks = [(rng.choice([1, 1, 2, 3, rng.randint(1, 60)]), rng.choice([3, 4])) for _ in range(rng.randint(1, 60))]
        starts, cost = [], 0
        for nt, unit in blocks:
            starts.append(cost)
            cost += nt * unit + ITEM
        n = min(148, -(-cost // 8))
        over = n % len(blocks)
        if over * 8 <= n and over < n:
            n -= over
        most = min(8, cost // n // 2)
        cuts = [i * cost // n for i in range(n + 1)]
        parts = [[] for _ in blocks]
        for i in range(n):
            begun = going_on = 0
            for b, (nt, unit) in enumerate(blocks):
                if starts[b] + nt * unit + ITEM <= cuts[i] or starts[b] >= cuts[i + 1]:
                    continue
                at = max(cuts[i], starts[b])
                j0, j1 = tile_at(at, starts[b], unit, nt, most), tile_at(cuts[i + 1], starts[b], unit, nt, most)
                if j0 < j1:
                    parts[b].append((i, j0, j1))
                    begun += j0 == 0 and j1 < nt
                    going_on += j0 > 0
            assert begun <= 1 and going_on <= 1  # two slots a CTA
        for b, (nt, unit) in enumerate(blocks):
            p = parts[b]
            assert p[0][1] == 0 and p[-1][2] == nt
            assert all(x[2] == y[1] and y[0] == x[0] + 1 for x, y in zip(p, p[1:]))
            # what the merge kernel counts, from the CTA that has the first part
            seen = [i for i in range(p[0][0], n) if tile_at(cuts[i], starts[b], unit, nt, most) <
                    tile_at(cuts[i + 1], starts[b], unit, nt, most)]
            assert len(p) == 1 or seen == [x[0] for x in p]
