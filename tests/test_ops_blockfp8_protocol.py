"""The FP8 product's barriers (csrc/ops_blockfp8.cu, many_rows) as a model on the CPU: who waits for whom, in random orders.

Threads are the copying one, the two that issue products, the tensor core and the scaling warps.  A thread carries what has
happened before it (a vector clock); a releasing arrive hands that to the barrier and a wait takes it, a relaxed arrive hands
over nothing.  A place of shared memory may be written by a copy only when all reads of what it held happened before.
"""

import random
import re

import pytest

from conftest import PKG

SOURCE = (PKG / "csrc" / "ops_blockfp8.cu").read_text()


def constant(name):
    return int(re.search(rf"\b{name} = (\d+)\b", SOURCE).group(1))


SCALES, RUN = constant("SCALES"), constant("SCALE_RUN")


def shape(bn, pair):
    """stages, buffers and scaling warps, as the kernel's ManyShape has them"""
    stage = 128 * 128 + (bn // 2 if pair else bn) * 128
    return 4 if stage > 40960 else 6 if stage >= 32768 else 8, min(4, 512 // bn), 8 if bn >= 128 else 4


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase, self.clock = 0, {}

    def arrive(self, clock):
        join(self.clock, clock)
        self.left -= 1
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def passed(self, parity):
        return self.phase % 2 != parity


def join(a, b):
    for k, v in b.items():
        a[k] = max(a.get(k, 0), v)


class Race(Exception):
    pass


class UnderWay(Exception):
    pass


def run(tiles, bn, pair, seed, hand_back=True, late=None, drain="whenever a wait gave up"):
    """``tiles``: the blocks of each tile that this block of threads takes.  Ends, or raises Race or a deadlock's AssertionError.

    ``late``: the block whose copies arrive after the limit of the waits only.  Then some wait gives up, all others learn of it, and
    what is under way is waited for (``drain``) before the block of threads ends: else UnderWay."""
    stages, buffers, warps = shape(bn, pair)
    full, empty = [Barrier(1) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    summed, read = [Barrier(1) for _ in range(buffers)], [Barrier(warps) for _ in range(buffers)]
    scaled = [Barrier(warps) for _ in range(SCALES // RUN)]
    reads = [dict() for _ in range(SCALES)]             # of a place: by whom, and when
    holds = [None] * SCALES
    blocks = sum(tiles)
    queue = []                                          # products and arrivals of the tensor core, in order
    flight = []                                         # copies under way
    gave_up = []

    def copies(me):
        stage = slot = 0
        phase = slot_phase = 0
        for i in range(blocks):
            yield empty[stage], phase ^ 1
            if hand_back and slot % RUN == 0:
                yield scaled[slot // RUN], slot_phase ^ 1
            for warp, when in reads[slot].items():
                if me["clock"].get(warp, 0) < when:
                    raise Race(f"block {i} overwrites scales that {warp} may still read")
            reads[slot], holds[slot] = {}, i
            flight.append((i, stage))
            slot += 1
            if slot == SCALES:
                slot, slot_phase = 0, slot_phase ^ 1
            stage += 1
            if stage == stages:
                stage, phase = 0, phase ^ 1

    def products(first):
        def go(me):
            stage = buffer = first
            phase = buffer_phase = 0
            for i in range(first, blocks, 2):
                yield read[buffer], buffer_phase ^ 1
                yield full[stage], phase
                queue.append((summed[buffer], dict(me["clock"])))
                if i < blocks - stages:
                    queue.append((empty[stage], dict(me["clock"])))
                stage += 2
                if stage >= stages:
                    stage, phase = stage - stages, phase ^ 1
                buffer += 2
                if buffer >= buffers:
                    buffer, buffer_phase = buffer - buffers, buffer_phase ^ 1
        return go

    def scaling(me):
        buffer = slot = phase = 0
        for i in range(blocks):
            yield summed[buffer], phase
            assert holds[slot] == i, "the scales of another block"
            me["clock"][me["name"]] = me["clock"].get(me["name"], 0) + 1
            reads[slot][me["name"]] = me["clock"][me["name"]]
            if hand_back and slot % RUN == RUN - 1:
                scaled[slot // RUN].arrive(me["clock"])         # releases
            slot = (slot + 1) % SCALES
            read[buffer].arrive({})                             # relaxed
            buffer += 1
            if buffer == buffers:
                buffer, phase = 0, phase ^ 1

    rng = random.Random(seed)
    threads = []
    for name, body in [("copies", copies), ("even", products(0)), ("odd", products(1))] + [(f"warp {w}", scaling) for w in range(warps)]:
        me = {"name": name, "clock": {}}
        threads.append([me, body(me), None])
    slow = rng.choice([t[0]["name"] for t in threads] + [None])         # one thread that lags behind
    while threads or queue:
        landing = [f for f in flight if f[0] != late]
        moves = [t for t in threads if t[2] is None or t[2][0].passed(t[2][1])]
        if queue:
            moves.append(None)
        if landing and (not moves or rng.random() < 0.5):
            f = rng.choice(landing)
            flight.remove(f)
            full[f[1]].arrive({})
            continue
        if not moves and late is not None:              # the limit passes: one thread gives up, the others that wait learn of it
            gave_up.extend(rng.sample([t[0]["name"] for t in threads], len(threads)))
            threads.clear()
            break
        assert moves, "deadlock"
        ready = [t for t in moves if t is None or t[0]["name"] != slow] or moves
        t = rng.choice(ready if rng.random() < 0.9 else moves)
        if t is None:
            barrier, clock = queue.pop(0)
            barrier.arrive(clock)
            continue
        if t[2] is not None:
            join(t[0]["clock"], t[2][0].clock)
        try:
            t[2] = next(t[1])
        except StopIteration:
            threads.remove(t)
    # every thread is at the block's last barrier: products under way are waited for by those who issued them
    while queue:
        barrier, clock = queue.pop(0)
        barrier.arrive(clock)
    if drain == "whenever a wait gave up" and gave_up or drain == "where the copies gave up" and "copies" in gave_up:
        for f in flight:
            full[f[1]].arrive({})
        flight.clear()
    if flight:
        raise UnderWay(f"copies of blocks {sorted(b for b, _ in flight)} arrive in memory that is no longer the block's")
    return gave_up


SHAPES = [(32, False), (64, False), (128, False), (256, True)]


@pytest.mark.parametrize("bn,pair", SHAPES)
@pytest.mark.parametrize("tiles", [[1], [3], [16], [17], [64, 64], [5, 5, 5, 5, 5], [1] * 40, [112, 3, 31]])
def test_scales_are_read_before_they_are_overwritten(bn, pair, tiles):
    for seed in range(20):
        run(tiles, bn, pair, seed)


@pytest.mark.parametrize("bn,pair", SHAPES)
def test_the_model_sees_a_missing_hand_back(bn, pair):
    with pytest.raises(Race):
        run([64], bn, pair, 0, hand_back=False)


@pytest.mark.parametrize("bn,pair", SHAPES)
def test_copies_never_wait_for_a_run(bn, pair):
    """The ring is long enough that its own barriers hold no copy up: what the other barriers allow lies in earlier runs."""
    stages, buffers, _ = shape(bn, pair)
    assert stages + buffers <= SCALES - RUN and SCALES % RUN == 0


@pytest.mark.parametrize("bn,pair", SHAPES)
@pytest.mark.parametrize("blocks,late", [(1, 0), (3, 2), (16, 0), (64, 40), (64, 63), (64, 60)])
def test_a_late_copy_ends_the_block_with_nothing_under_way(bn, pair, blocks, late):
    for seed in range(20):
        assert run([blocks], bn, pair, seed, late=late)


@pytest.mark.parametrize("bn,pair", SHAPES)
def test_the_model_sees_a_copy_that_nobody_waits_for(bn, pair):
    """The last copies: the thread that issued them is done and did not give up itself."""
    with pytest.raises(UnderWay):
        run([64], bn, pair, 0, late=63, drain="where the copies gave up")
