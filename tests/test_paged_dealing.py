"""How attention over a paged cache deals its work out, modelled step by step (CPU): every block of every tile is taken once, and
the join reads the partial rows that were written, over batches of any number of sequences."""

from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

import thundersync_amd

SOURCE = (Path(thundersync_amd.__file__).parent / "csrc" / "paged_attention.h").read_text()
BLOCK, COST = map(int, re.search(r"kBlockKeys = (\d+), kTileCost = (\d+);", SOURCE).groups())
SNAP = int(re.search(r"kSnap = (\d+);", SOURCE).group(1))
LEAST = tuple(map(int, re.search(r"kLeast = KERNEL == 0 \? (\d+) : (\d+);", SOURCE).groups()))


def snapped(border, inside, blocks):
    """Where a border `inside` blocks within a tile goes."""
    if 2 * inside <= blocks:
        return border - inside if inside < SNAP else border
    return border + blocks - inside if blocks - inside < SNAP else border


class Batch:
    """Sequences as (tiles, blocks of each tile); the work of one KV head."""

    def __init__(self, seqs, jobs, least):
        self.seqs, self.total = seqs, sum(t * b for t, b in seqs)
        self.per = max(-(-self.total // jobs), least)
        self.used = -(-self.total // self.per)

    def begin(self, job):
        """(sequence, tile, block in it, first block, end) of a work-group, or None: two borders found over 64 sequences at a time."""
        if job >= self.used:
            return None
        borders = job * self.per, min((job + 1) * self.per, self.total)
        start, stop, before, found = 0, self.total if borders[1] == self.total else 0, 0, None
        for s0 in range(0, len(self.seqs), 64):
            upto, at = [], before
            for tiles, blocks in self.seqs[s0:s0 + 64]:
                at += tiles * blocks
                upto.append(at)
            for k in (0, 1):
                if not before <= borders[k] < at:
                    continue
                lane = next(i for i, u in enumerate(upto) if u > borders[k])
                tiles, size = self.seqs[s0 + lane]
                nth, x = divmod(borders[k] - (upto[lane] - tiles * size), size)
                to = snapped(borders[k], x, size)
                if k:
                    stop = to
                else:
                    start, found = to, [s0 + lane, nth, x + to - borders[k]]
            if found and stop > 0:
                break
            before = at
        if not found or stop <= start:
            return None
        s, tile, block = found
        if block == self.seqs[s][1]:
            tile, block = tile + 1, 0
            if tile >= self.seqs[s][0]:
                s, tile = self.skip(s), 0
                if s is None:
                    return None
        return s, tile, block, start, stop

    def skip(self, s):
        return next((i for i in range(s + 1, len(self.seqs)) if self.seqs[i][0]), None)

    def pieces(self, job):
        """(sequence, tile, from, to, first block of the tile if the work-group begins it)"""
        place = self.begin(job)
        if place is None:
            return
        s, tile, block, start, stop = place
        left = stop - start
        while True:
            blocks = self.seqs[s][1]
            yield s, tile, block, min(blocks, block + left), stop - left if block == 0 else None
            left -= min(blocks, block + left) - block
            if left <= 0:
                return
            tile, block = tile + 1, 0
            if tile >= self.seqs[s][0]:
                s, tile = self.skip(s), 0
                if s is None:
                    return

    def parts(self, start, tile, blocks):
        """The slots that the join reads of a tile, in order, of a sequence whose first tile begins at `start`."""
        first = start + tile * blocks
        last = first + blocks
        owner, inner = (first + min(SNAP - 1, blocks // 2)) // self.per, (first + SNAP + self.per - 1) // self.per
        n = 1 + max(0, (last - SNAP) // self.per - inner + 1)
        return [2 * owner + 1] + [2 * (inner + p - 1) for p in range(1, n)]


def check(seqs, jobs, least):
    batch = Batch(seqs, jobs, least)
    taken, starts = {}, {}
    for job in range(batch.used):
        for s, tile, a, b, start in batch.pieces(job):
            taken.setdefault((s, tile), []).append((a, b, 2 * job + (a == 0)))
            if start is not None and tile == 0:
                assert s not in starts
                starts[s] = start
    assert batch.used <= jobs
    at = 0
    for s, (tiles, blocks) in enumerate(seqs):
        if tiles:
            assert starts[s] == at
        for tile in range(tiles):
            runs = taken.pop((s, tile))
            assert runs[0][0] == 0 and runs[-1][1] == blocks and all(x[1] == y[0] for x, y in zip(runs, runs[1:]))
            assert all(a < b for a, b, _ in runs)
            assert [slot for *_, slot in runs] == batch.parts(at, tile, blocks)
        at += tiles * blocks
    assert not taken


def draw(rng):
    n = rng.choice((1, 2, 5, 63, 64, 65, 128, 129, 200, 300))
    longest = rng.choice((1, 3, 20, 120, 1000))
    shortest = rng.choice((0, 0, longest))
    many = rng.choice((1, 1, 2, 40))
    idle = rng.choice((0.0, 0.1, 0.9))
    return [(0 if rng.random() < idle else rng.randint(1, many), COST + rng.randint(shortest, longest)) for _ in range(n)]


@pytest.mark.parametrize("least", LEAST)
def test_every_block_is_taken_once_and_found_by_the_join(least):
    rng = random.Random(least)
    for _ in range(400):
        check(draw(rng), rng.choice((1, 2, 7, 32, 64, 96, 256, 768)), least)


@pytest.mark.parametrize("jobs", [1, 2, 63, 64, 96, 256, 768])
@pytest.mark.parametrize("n", [64, 65, 128, 129, 131, 256])
def test_borders_beyond_the_first_64_sequences(n, jobs):
    """The last work-groups' end is known before their beginning is found."""
    for blocks in range(COST, COST + 24):
        check([(1, blocks)] * n, jobs, LEAST[0])
        check([(3, blocks)] * n, jobs, LEAST[1])


def test_a_search_that_stops_at_the_first_border_is_seen():
    """The model shows a work-group that finds its end and not its beginning."""

    class Short(Batch):
        def begin(self, job):
            seqs, self.seqs = self.seqs, self.seqs[:64] if (job + 1) * self.per >= self.total else self.seqs
            try:
                return super().begin(job)
            finally:
                self.seqs = seqs

    batch = Short([(1, COST + 20)] * 130, 96, LEAST[0])
    assert list(batch.pieces(batch.used - 1)) == [] and list(Batch(batch.seqs, 96, LEAST[0]).pieces(batch.used - 1)) != []
