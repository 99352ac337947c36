"""The dense products' LDS ring over several tiles, simulated on the CPU.

dense_tile (cuda-moe-engine_amd/csrc/linear_ring.h) waits for counts of vector memory operations, which complete in
issue order: the loads of the windows ahead, and between two tiles the first one's stores, which go out after all of the
next tile's first loads. A wait is right when no load of the stage that is read next is among the operations it leaves out.
This replays the issue order tile after tile, chained or not, with the stores that an epilogue is sure to issue (and with
more of them), and checks each stage's loads before its first read and each slot before its refill. The depths and counts
are the kernel's.
"""

import itertools

import pytest

LINE = 128


def depths(tm, bn, lds, cap=6):
    a, b = tm * LINE, bn * LINE
    equal = min(lds // (a + b), cap)
    return (equal, equal) if equal >= 3 else (2, (lds - 2 * a) // b)


class Ring:
    def __init__(self, tm, bn, kib, chained_stores):
        self.sa, self.sb = depths(tm, bn, kib * 1024)
        assert 2 <= self.sa <= self.sb and self.sa * tm * LINE + self.sb * bn * LINE <= kib * 1024
        self.a_loads, self.b_loads = tm // 32, bn // 32
        loads = self.a_loads + self.b_loads
        self.steady = (self.b_loads if self.sb > self.sa else 0) + (self.sa - 2) * loads
        self.first = (self.b_loads if self.sb > self.sa else 0) + (self.sa - 1) * loads
        self.stores = chained_stores
        assert self.first + self.stores < 64
        self.queue = []   # operations in flight, oldest first
        self.slots = {}   # (matrix, slot) -> (tile, stage) that lies or lands there
        self.read = set()  # (matrix, tile, stage) whose last read is behind a barrier

    def load(self, matrix, tile, stage, slot, real):
        before = self.slots.get((matrix, slot))
        assert before is None or before == (tile, stage) or (matrix, *before) in self.read, (matrix, tile, stage)
        self.slots[matrix, slot] = (tile, stage)
        self.queue += [(matrix, tile, stage, real)] * (self.a_loads if matrix == "a" else self.b_loads)

    def wait(self, count):
        del self.queue[: max(len(self.queue) - count, 0)]

    def use(self, tile, stage, sa, sb):
        assert self.slots["a", sa] == (tile, stage) and self.slots["b", sb] == (tile, stage)
        assert not any(op[0] in "ab" and op[1:3] == (tile, stage) for op in self.queue), (tile, stage)


def prologue(ring, tile, steps, a0, b0, chained):
    for v in range(-ring.sb, 0):
        if chained and v != -1:
            continue
        if v + ring.sa >= 0:
            load_clamped(ring, "a", tile, v + ring.sa, (a0 + v) % ring.sa, steps)
        load_clamped(ring, "b", tile, v + ring.sb, (b0 + v) % ring.sb, steps)


def load_clamped(ring, matrix, tile, stage, slot, steps):
    # Stages past the end load the last one again into a slot that nothing reads: the tag keeps them apart.
    ring.load(matrix, tile, stage if stage < steps else (stage, "again"), slot, stage < steps)


def run(tm, bn, kib, steps_of_tiles, stores, issued_stores):
    ring = Ring(tm, bn, kib, stores)
    sa0 = sb0 = 0
    prologue(ring, 0, steps_of_tiles[0], 0, 0, False)
    for t, steps in enumerate(steps_of_tiles):
        after = t > 0
        following = steps_of_tiles[t + 1] if t + 1 < len(steps_of_tiles) else None
        chain = following is not None and steps >= ring.sb and following >= ring.sb
        na, nb = (sa0 + steps) % ring.sa, (sb0 + steps) % ring.sb
        slack = stores if after else 0
        ring.wait(ring.first + slack)
        ring.use(t, 0, sa0, sb0)
        sa, sb = sa0, sb0
        for u in range(steps - 1):
            ring.wait(ring.steady + (slack if u == 0 else 0))
            ring.read |= {("a", t, u), ("b", t, u)}  # its fragments are in registers on every wave
            na_u, nb_u = (sa + 1) % ring.sa, (sb + 1) % ring.sb
            for matrix, depth, slot in (("a", ring.sa, sa), ("b", ring.sb, sb)):
                stage = u + depth
                if chain and stage >= steps:
                    ring.load(matrix, t + 1, stage - steps, slot, True)
                else:
                    load_clamped(ring, matrix, t, stage, slot, steps)
            sa, sb = na_u, nb_u
            ring.use(t, u + 1, sa, sb)
        ring.wait(0)
        # Every wave is past the tile's last read; repeated loads are read by no one.
        ring.read |= {("a", t, steps - 1), ("b", t, steps - 1)}
        ring.read |= {(m, *ring.slots[m, s]) for m, s in ring.slots if isinstance(ring.slots[m, s][1], tuple)}
        if following is not None:
            if not chain:
                ring.slots.clear()
            prologue(ring, t + 1, following, na if chain else 0, nb if chain else 0, chain)
            ring.queue += [("store",)] * issued_stores
            sa0, sb0 = (na, nb) if chain else (0, 0)


@pytest.mark.parametrize("swiglu", [False, True])
def test_chained_tiles_of_256(swiglu):
    stores = 8 * (4 if swiglu else 8) // 2
    for steps in itertools.product((1, 2, 3, 4, 7, 32), repeat=3):
        for issued in (stores, stores + 5, 3 * stores):
            run(256, 256, 160, steps, stores, issued)


def test_a_wait_that_leaves_out_more_stores_than_there_are_is_found():
    with pytest.raises(AssertionError):
        run(256, 256, 160, (8, 8), 32, 0)


@pytest.mark.parametrize("tm,bn,kib", [(64, 64, 80), (64, 128, 80), (96, 128, 80), (128, 128, 80), (128, 128, 160)])
def test_single_tiles(tm, bn, kib):
    for steps in range(1, 40):
        run(tm, bn, kib, (steps,), 0, 0)
