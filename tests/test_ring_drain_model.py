"""Host model of how the producers of the 4-bit kernels end (fp4_common.cuh::drain_ring): every copy that a producer has issued has
landed when it leaves, and no wait is one for a phase that never comes."""
import re
from pathlib import Path

import pytest

KERNELS = Path(__file__).resolve().parent.parent / "csrc" / "kernels"


def looked_at(stages, s, round_, step, ok):
    """(stage, round) pairs that the producer waits for, as the kernel counts them."""
    out, issued = [], (round_ * stages + s) // step
    for i in range(min(issued, (stages + (0 if ok else step - 1)) // step)):
        s -= step
        if s < 0:
            s, round_ = s + stages, round_ - 1
        out.append((s, round_))
    return out


def place(block, stages):
    return block % stages, block // stages


@pytest.mark.parametrize("stages", range(3, 13))
@pytest.mark.parametrize("producers", [1, 2])
def test_every_copy_in_flight_and_no_phase_that_never_comes(stages, producers):
    for blocks in range(0, 4 * stages + 3):
        for mine in range(producers):
            own = list(range(mine, blocks, producers))
            nxt = own[-1] + producers if own else mine
            waits = looked_at(stages, *place(nxt, stages), producers, True)
            last = {}                                    # the last round that any producer issues into a stage
            for b in range(blocks):
                last[b % stages] = b // stages
            # a parity wait for round r passes once r is complete and until r + 1 is: no later round may complete
            assert all(last[s] == r for s, r in waits)
            assert [place(b, stages) for b in reversed(own)][:len(waits)] == waits
            # what is not looked at was consumed before its stage's next block, or lies one place too far back of an odd ring
            rest = [b for b in own if place(b, stages) not in waits and last[b % stages] == b // stages]
            assert len(rest) <= (stages % 2 if producers == 2 else 0)
            failed = looked_at(stages, *place(nxt, stages), producers, False)
            assert failed[:len(waits)] == waits and all(place(b, stages) in failed for b in rest)


def test_each_producer_ends_with_it():
    for name, n in (("fp4_gemm.cu", 2), ("fp4_moe.cu", 2)):
        text = re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())
        assert len(re.findall(r"drain_ring\(full\(0\)", text)) == n
