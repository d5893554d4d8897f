"""The few-token fp8 kernel's schedule played through on the CPU: producer, two issuers, tensor cores, scale warps and
epilogue as agents that meet at barriers like the kernel's (csrc/gemm_f8_tc.cu, gemm_f8_few_kernel), in random order.

A barrier completes a phase when as many have arrived as it counts; waiting for a parity ends when the phase of that
parity is the last complete one.  So a wait that is a whole two phases behind passes wrongly, which is what the checks
of the contents would show.
"""

import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count, self.arrived, self.phases = count, 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.arrived, self.phases = 0, self.phases + 1

    def passed(self, parity):
        return (self.phases - 1) % 2 == parity  # before the first phase: as if one of parity 1 were complete


def play(stages, per_stage, accumulators, blocks, tiles, seed):
    """One block's share: `tiles` tiles of `blocks` K blocks, `per_stage` of them a stage."""
    rng = random.Random(seed)
    slots = 4
    full, empty = [Barrier(1) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    sums_full, sums_empty = [Barrier(2) for _ in range(2)], [Barrier(4) for _ in range(2)]
    scales_full, scales_empty = [Barrier(4) for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    ring, scales, sums, finished = [None] * stages, [None] * slots, {}, []
    queue, copies = [], []  # what the tensor cores and the copy engine have been given

    def producer():
        s = phase = 0
        for tile in range(tiles):
            for kb in range(0, blocks, per_stage):
                while not empty[s].passed(phase ^ 1):
                    yield
                ring[s] = None  # the copy is on its way
                copies.append((s, (tile, kb)))
                yield
                s += 1
                if s == stages:
                    s, phase = 0, phase ^ 1

    def copier():
        while True:
            if copies:
                s, what = copies.pop(rng.randrange(len(copies)))  # copies may land in any order
                ring[s] = what
                full[s].arrive()
            yield

    def tensor_cores():
        while True:
            if queue:
                op, *args = queue.pop(0)
                if op == "commit":
                    args[0].arrive()
                else:
                    s, slot, buf, which, tile, kb, first = args
                    assert ring[s] == (tile, kb - kb % per_stage), "operands"
                    assert scales[slot] == (tile, kb - kb % 4), "scales"
                    if first:
                        sums[buf, which] = []
                    sums[buf, which].append((tile, kb))
            yield

    def issuer(which):
        s, phase, slot = which, 0, 0
        for tile in range(tiles):
            buf = tile % accumulators
            while not sums_empty[buf].passed(((tile // accumulators) & 1) ^ 1):
                yield
            first = (which ^ ((tile * -(-blocks // per_stage)) & 1)) * per_stage
            any_yet = False
            for kb in range(0, blocks, 4):
                while not scales_full[slot % slots].passed((slot // slots) & 1):
                    yield
                for h0 in range(0, 4, 2 * per_stage):
                    h = h0 + first
                    if kb + h >= blocks:
                        break
                    while not full[s].passed(phase):
                        yield
                    for i in range(per_stage):
                        if kb + h + i < blocks:
                            queue.append(("mma", s, slot % slots, buf, which, tile, kb + h + i, not any_yet))
                            any_yet = True
                        yield
                    queue.append(("commit", empty[s]))
                    s += 2
                    if s >= stages:
                        s, phase = which, phase ^ 1
                queue.append(("commit", scales_empty[slot % slots]))
                slot += 1
                yield
            queue.append(("commit", sums_full[buf]))

    def scale_warps():
        slot = 0
        for tile in range(tiles):
            for kb in range(0, blocks, 4):
                while not scales_empty[slot % slots].passed(((slot // slots) & 1) ^ 1):
                    yield
                scales[slot % slots] = (tile, kb)
                yield
                for _ in range(4):
                    scales_full[slot % slots].arrive()
                slot += 1

    def epilogue():
        for tile in range(tiles):
            buf = tile % accumulators
            while not sums_full[buf].passed((tile // accumulators) & 1):
                yield
            # a tile of one stage has sums in the accumulator of the issuer whose turn it was
            one = (tile * -(-blocks // per_stage)) & 1
            which = (0, 1) if blocks > per_stage else (one,)
            got = sorted(p for w in which for p in sums[buf, w])
            assert got == [(tile, kb) for kb in range(blocks)], "sums"
            yield
            assert sorted(p for w in which for p in sums[buf, w]) == got, "sums overwritten"
            finished.append(tile)
            for _ in range(4):
                sums_empty[buf].arrive()

    agents = [producer(), issuer(0), issuer(1), scale_warps(), epilogue()]
    engines = [copier(), tensor_cores()]
    for _ in range(400 * tiles * (blocks + 8) * 7):
        if not agents:
            break
        a = rng.choice(agents + engines)
        try:
            next(a)
        except StopIteration:
            agents.remove(a)
    assert not agents, "an agent waits for good"
    assert finished == list(range(tiles))


@pytest.mark.parametrize("per_stage,accumulators", [(1, 1), (2, 2)])  # tiles of 128 tokens, and smaller ones
@pytest.mark.parametrize("stages", [2, 4, 6, 8])
def test_schedule(stages, per_stage, accumulators):
    for blocks in (1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 23, 33):
        for seed in range(2):
            play(stages, per_stage, accumulators, blocks, 5, seed)


def test_an_odd_ring_would_be_noticed():
    # two issuers that take every other stage of three
    with pytest.raises(AssertionError):
        for seed in range(20):
            play(3, 2, 2, 9, 5, seed)
