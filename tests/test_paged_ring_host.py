"""CPU: the ring of K and V copies in paged_prompt.cu. A barrier tells a phase only from the one before, so a warp that waits
for the same slot's next copy while two of them are done waits for good. The arrivals that the source gives `free` are put into
a model of the ring in which one warp at a time is held back as long as the others let it: it must not miss a copy."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "-1.7-atlas---apollo_b200", "csrc", "paged_prompt.cu")


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0, "more arrivals than the barrier counts"
        if not self.left:
            self.left, self.phase = self.count, self.phase + 1

    def done(self, use):
        """What a wait for copy number `use` of the slot sees: only the phase's parity."""
        assert self.phase - use <= 1, "a phase has passed that this warp still waits for"
        return self.phase % 2 != use % 2


def _source():
    text = open(SOURCE).read()
    const = {n: int(v) for n, v in re.findall(r"\b(k\w+) = (\d+)u?[,;]", text)}
    init = re.search(r"mbar_init\(&b\.free\[i\], ([^)]+)\)", text).group(1)
    count = eval(re.sub(r"(\d)u", r"\1", init), {}, const)
    checks = text[text.index("- checks --"):text.index("- softmax --")]
    return const["kCheckers"], count, "mbar_arrive(&b.free[" in checks


def _run(stages, copies, held, checkers, count, checkers_arrive):
    """The producer, the MMA warp and the checkers over `copies` copies; `held` moves only where nothing else can."""
    full, free = [Barrier(1) for _ in range(stages)], [Barrier(count) for _ in range(stages)]

    def producer():
        for n in range(copies):
            while n >= stages and not free[n % stages].done(n // stages - 1):
                yield False
            full[n % stages].arrive()
            yield True

    def consumer(arrives):
        for n in range(copies):
            while not full[n % stages].done(n // stages):
                yield False
            if arrives:
                free[n % stages].arrive()
            yield True

    warps = [producer(), consumer(True)] + [consumer(checkers_arrive) for _ in range(checkers)]
    going = set(range(len(warps)))
    while going:
        moved = False
        for i in sorted(going, key=lambda i: i == held):   # the one that is held back comes last
            if i == held and moved:
                continue
            step = next(warps[i], None)
            if step is None:
                going.discard(i)
            moved |= step is not False
        assert moved, "every warp waits"


@pytest.mark.parametrize("stages", [5, 6])
@pytest.mark.parametrize("held", [0, 1, 2, 3])
def test_no_warp_misses_a_copy(stages, held):
    checkers, count, arrive = _source()
    _run(stages, 40 * stages + 3, held, checkers, count, arrive)
