"""The ring protocol of the shared-prefix kernel (csrc/prefix_attend.cu) as a model: which role waits for which
phase of which barrier.  Barriers have the hardware's semantics (a wait sees only the parity of the current
phase, an arrival too many is an error) and loads land in any order.  Checked: every product finds its own tile,
scales are not overwritten while they are used, every role finishes."""
import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = self.bytes = 0

    def arrive(self):
        assert self.pending > 0, "an arrival too many"
        self.pending -= 1
        self.settle()

    def settle(self):
        if self.pending == 0 and self.bytes == 0:
            self.phase += 1
            self.pending = self.count

    def passed(self, parity):
        return (self.phase & 1) != parity


def simulate(tiles, pair, codes, rng, rate):
    stride = 1 if pair else 2
    stages = (3 if codes else 5) + (0 if pair else 1)
    per_stream = stages if pair else stages // 2
    raw_stages = 3

    def index_of(j, v):
        return 2 * (j if pair else j >> 1) + v

    def stage_of(j, v):
        return index_of(j, v) % per_stream + (0 if pair else (j & 1) * per_stream)

    def round_of(j, v):
        return (index_of(j, v) // per_stream) & 1

    def tiles_of(stream):
        return list(range(tiles)) if pair else list(range(stream, tiles, 2))

    order = []
    for j in range(-stride, tiles):
        order += ([(j, 1)] if j >= 0 else []) + ([(j + stride, 0)] if j + stride < tiles else [])
    full, empty = [Barrier(1) for _ in range(stages)], [Barrier(2 if pair else 1) for _ in range(stages)]
    raw_full, raw_empty = [Barrier(1) for _ in range(raw_stages)], [Barrier(1) for _ in range(raw_stages)]
    s_full, p_full, turn = ([Barrier(1) for _ in range(2)] for _ in range(3))
    scales_full = [Barrier(1) for _ in range(4)]
    data, raw, scale, weighted, flying = [None] * stages, [None] * raw_stages, [None] * 4, set(), []

    def producer():
        for n, (j, v) in enumerate(order):
            if codes:
                s, rd, f, e, place = n % raw_stages, (n // raw_stages) & 1, raw_full, raw_empty, raw
            else:
                s, rd, f, e, place = stage_of(j, v), round_of(j, v), full, empty, data
            while not e[s].passed(rd ^ 1):
                yield
            place[s] = None
            f[s].bytes += 1
            f[s].arrive()
            flying.append((f[s], place, s, (j, v)))
            yield

    def converter():
        n = 0
        for j in range(-stride, tiles):
            jk = j + stride
            both = ([(j, 1)] if j >= 0 else []) + ([(jk, 0)] if jk < tiles else [])
            for at, (t, v) in enumerate(both, n):
                while not raw_full[at % raw_stages].passed((at // raw_stages) & 1):
                    yield
                while not empty[stage_of(t, v)].passed(round_of(t, v) ^ 1):
                    yield
            for t, v in both:
                assert raw[n % raw_stages] == (t, v)
                raw[n % raw_stages] = None
                raw_empty[n % raw_stages].arrive()
                n += 1
                data[stage_of(t, v)] = (t, v)
                yield
            for t, v in both:
                full[stage_of(t, v)].arrive()
            if jk < tiles:
                users = (0, 1) if pair else (jk % 2,)
                assert jk < 4 or all((s, jk - 4) in weighted for s in users), "scales in use"
                scale[jk % 4] = jk
                scales_full[jk % 4].arrive()
            yield

    def products(stream):
        mine = tiles_of(stream)

        def scores(j):
            assert data[stage_of(j, 0)] == (j, 0), "another K tile"
            empty[stage_of(j, 0)].arrive()
            s_full[stream].arrive()
        for k, j in enumerate(mine):
            if k == 0:
                while not full[stage_of(j, 0)].passed(round_of(j, 0)):
                    yield
                scores(j)
                yield
            ahead = mine[k + 1:k + 2]
            for t, v in [(j, 1)] + [(a, 0) for a in ahead]:
                while not full[stage_of(t, v)].passed(round_of(t, v)):
                    yield
            while not p_full[stream].passed(k & 1):
                yield
            assert data[stage_of(j, 1)] == (j, 1), "another V tile"
            empty[stage_of(j, 1)].arrive()
            yield
            for a in ahead:
                scores(a)
            yield

    def softmax(stream):
        for k, j in enumerate(tiles_of(stream)):
            while not s_full[stream].passed(k & 1):
                yield
            while codes and not scales_full[j % 4].passed((j // 4) & 1):
                yield
            while (stream or k) and not turn[stream].passed((k if stream else k - 1) & 1):
                yield
            yield
            assert not codes or scale[j % 4] == j, "another tile's scales"
            turn[1 - stream].arrive()
            weighted.add((stream, j))
            p_full[stream].arrive()
            yield

    roles = [producer(), products(0), products(1), softmax(0), softmax(1)] + ([converter()] if codes else [])
    idle = 0
    while roles and idle < 50000:
        idle += 1
        if flying and rng.random() < rate:
            bar, place, s, what = flying.pop(rng.randrange(len(flying)))
            place[s] = what
            bar.bytes -= 1
            bar.settle()
            idle = 0
        role = rng.choice(roles)
        try:
            next(role)
        except StopIteration:
            roles.remove(role)
            idle = 0
    assert not roles and not flying, "a role waits for good"


@pytest.mark.parametrize("codes", [False, True])
@pytest.mark.parametrize("pair", [False, True])
def test_every_product_finds_its_tile_and_every_role_ends(pair, codes):
    rng = random.Random(5)
    for tiles in (1, 2, 3, 4, 5, 7, 9, 18):
        for rate in (0.3, 0.05):
            for _ in range(12):
                simulate(tiles, pair, codes, rng, rate)
