"""Host model of the weight ring of the 4-bit expert kernels: two producers that take every other block and one consumer that
waits for two stages at a time, on mbarriers with phase parities.  No wait may pass before the phase it means."""
import random

import pytest


class Barrier:
    """One arrival per phase; a parity wait passes when the current phase's parity differs from the one waited for."""

    def __init__(self):
        self.phase = 0

    def passes(self, parity):
        return (self.phase & 1) != parity

    def arrive(self):
        self.phase += 1


def run(stages, blocks, seed, delays):
    rng = random.Random(seed)
    full, empty = [Barrier() for _ in range(stages)], [Barrier() for _ in range(stages)]
    holds = [None] * stages      # block whose copy was issued into the stage
    landing = []                 # (stage, block) copies in flight
    freeing = []                 # stages whose MMAs were issued, in order
    used = []
    prod = [{"it": p, "s": p % stages, "round": p // stages} for p in (0, 1)]
    cons = {"it": 0, "s": 0, "par": 0}
    for _ in range(200000):
        if len(used) == blocks and not freeing:
            break
        who = rng.choices(("p0", "p1", "c", "land", "free"), weights=delays)[0]
        if who in ("p0", "p1"):
            p = prod[who == "p1"]
            if p["it"] < blocks and (p["round"] == 0 or empty[p["s"]].passes((p["round"] - 1) & 1)):
                s = p["s"]
                # the stage's last block was consumed and its MMAs are complete
                assert holds[s] is None, ("overwrote", holds[s], "with", p["it"])
                holds[s] = p["it"]
                landing.append((s, p["it"]))
                p["it"] += 2
                p["s"] += 2
                if p["s"] >= stages:
                    p["s"] -= stages
                    p["round"] += 1
        elif who == "land" and landing:
            s, b = landing.pop(rng.randrange(len(landing)))   # copies complete in any order
            full[s].arrive()
        elif who == "c" and cons["it"] < blocks:
            two = cons["it"] + 1 < blocks
            s, par = cons["s"], cons["par"]
            s1, par1 = (0, par ^ 1) if s + 1 == stages else (s + 1, par)
            if full[s].passes(par) and (not two or full[s1].passes(par1)):
                for k, st in enumerate((s, s1)[:1 + two]):
                    assert holds[st] == cons["it"] + k and (st, holds[st]) not in landing, "read a stage that is not its block's"
                    used.append(holds[st])
                    freeing.append(st)
                cons["it"] += 1 + two
                if two:
                    s, par = s1, par1
                cons["s"], cons["par"] = (0, par ^ 1) if s + 1 == stages else (s + 1, par)
        elif who == "free" and freeing:
            s = freeing.pop(0)                                # MMAs complete in order
            holds[s] = None
            empty[s].arrive()
    assert used == list(range(blocks))


@pytest.mark.parametrize("stages", [3, 4, 5, 7, 9, 10, 12])
@pytest.mark.parametrize("blocks", [1, 2, 3, 11, 40])
def test_no_wait_passes_early(stages, blocks):
    for seed in range(8):
        run(stages, blocks, seed, (1, 1, 1, 1, 1))
        run(stages, blocks, seed, (8, 1, 4, 4, 1))     # one producer far ahead, slow tensor core
        run(stages, blocks, seed, (1, 8, 1, 8, 8))
