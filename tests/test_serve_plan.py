"""How the attention against a cache is cut into parts: the host bounds the parts of a sequence (the workspace) and the
workgroups (the grid) without knowing the lengths; the device then picks the pages of a part from the lengths.  Both are
restated here and the bounds checked for every kind of batch: a part beyond the workspace would be written out of range, and one
beyond the grid would never run."""
import random

import pytest

CUS, SHORT_PART, LONG_PART, ROUNDS = 256, 48, 24, 4
LONG_GROUPS = ROUNDS * CUS


def host(B, units, pages, D, steps, page_bytes, prefix):
    nw = 8 if D <= 128 else 4
    least = max(nw // steps, 1)
    least = max(least, nw * (16 << 10) // page_bytes // least * least)
    slots = CUS // 4 if prefix else CUS
    items, every, cut = B * units, -(-pages // least), -(-pages // LONG_PART)
    nchunk = min(every, max(cut, max(slots // units, 1)) if items < slots else cut)
    if not prefix and pages <= 2 * least:
        nchunk = 1
    fullest = items * -(-pages // (48 * nw))
    groups = min(items * cut, max(LONG_GROUPS, fullest) + items)
    groups = min(max(groups, slots) if items < slots else groups, items * nchunk)
    return least, slots, nchunk, groups, 48 * nw


def device(lens, units, pages, least, slots, nchunk, most, prefix):
    B = len(lens)
    if nchunk == 1:
        return max(pages, 1)

    def count(c):
        return sum(max(-(-n // c), 1) for n in lens) * units
    work = sum(lens) * units
    floor = max(least, -(-pages // nchunk))
    if not prefix and max(lens) <= 2 * least:
        return max(2 * least, floor)
    c = max(min(-(-work // slots) + least - 1, SHORT_PART) // least * least, floor)
    for _ in range(10):
        if not (c < SHORT_PART and B * units < slots):
            break
        if count(c) <= slots:
            return c
        c = (c + c // 8 + least) // least * least
    for r in (1, 2, 4):
        c = min(most, max(LONG_PART, floor, -(-work // (r * CUS))))
        for k in range(4):
            if c >= most:
                break
            if count(c) <= r * CUS:
                return c
            if k < 3:
                c = min(c + (c + 23) // 24, most)
    return max(c, floor)


@pytest.mark.parametrize("seed", range(40))
def test_parts_stay_within_the_workspace_and_the_grid(seed):
    r = random.Random(seed)
    for _ in range(400):
        D = r.choice([16, 32, 64, 128, 256])
        size = r.choice([1, 2, 4])
        B, units = r.choice([1, 2, 3, 7, 16, 64, 300]), r.choice([1, 2, 5, 8, 12, 16, 40, 96])
        pages = max(1, int(2 ** r.uniform(0, 17 if B < 16 else 12)))
        steps, prefix = r.choice([1, 2, 4]), r.random() < 0.4
        least, slots, nchunk, groups, most = host(B, units, pages, D, steps, 2 * 64 * D * size, prefix)
        kind = r.choice(["full", "short", "ragged", "one"])
        lens = [pages if kind == "full" or (kind == "one" and b == 0) else r.randint(0, pages if kind == "ragged" else min(pages, 3))
                for b in range(B)]
        c = device(lens, units, pages, least, slots, nchunk, most, prefix)
        parts = [max(-(-n // c), 1) for n in lens]
        nw = 8 if D <= 128 else 4
        assert max(parts) <= nchunk
        assert sum(parts) * units <= groups, (sum(parts) * units, groups)
        # a wave keeps the page numbers of its share of a part in one register: 64 of them
        assert nchunk == 1 or -(-c // nw) + 1 <= 64
        assert nchunk > 1 or -(-pages // nw) + 1 <= 64
