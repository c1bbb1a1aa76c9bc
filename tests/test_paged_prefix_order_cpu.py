"""The tensor-core prefix's last waits, restated from the device code: one thread
issues the products, they run in the order of issue, the softmax of each query
tile runs beside them.  A wait for a barrier's phase of parity p returns when
the phase in progress has the other parity: too early while the phase before the
one that is meant is in progress, and never when the one after it is over."""
import random

import pytest


class Barrier:
    def __init__(self):
        self.phase = 0

    def passes(self, parity):
        return (self.phase & 1) != parity


def _issue(SB, MT, n, sfull, pfull, odone, queue):
    """What the issuing thread does: ("wait", barrier, parity) or appends to the queue."""
    def scores(m, t):
        queue.append(("S", m, t))
        queue.append(("commit", sfull[SB * m + t % SB]))
    for m in range(MT):
        scores(m, 0)
    for t in range(n):
        more = t + 1 < n
        if SB == 2 and more:
            scores(0, t + 1)
        for m in range(MT):
            yield pfull[SB * m + t % SB], (t // SB) & 1
            queue.append(("PV", m, t))
            queue.append(("commit", odone[m]))
            if SB == 1 and more:
                scores(m, t + 1)


def _softmax(SB, MT, m, n, sfull, pfull, odone, guard, moves):
    for t in range(n):
        yield sfull[SB * m + t % SB], (t // SB) & 1
        if t > 0 and moves():  # the reference moves: the sums so far are rescaled
            yield odone[m], (t - 1) & 1
        if guard and SB == 2 and t > 0 and t == n - 1:
            yield odone[m], (t - 1) & 1
        pfull[SB * m + t % SB].phase += 1
    for k in [m] + ([m ^ 1] if MT == 2 else []):
        yield odone[k], (n - 1) & 1


def _run(SB, MT, n, guard, rng):
    """True when every query tile leaves, and after all products have run."""
    sfull, pfull = ([Barrier() for _ in range(4)] for _ in range(2))
    odone = [Barrier() for _ in range(2)]
    queue, done = [], 0
    actors = {"issue": _issue(SB, MT, n, sfull, pfull, odone, queue)}
    for m in range(MT):
        actors[m] = _softmax(SB, MT, m, n, sfull, pfull, odone, guard,
                             lambda: rng.random() < 0.1)
    waits = {k: next(a, None) for k, a in actors.items()}
    speed = {k: rng.choice([1, 4, 16]) for k in list(actors) + ["run"]}
    while True:
        ready = [k for k, w in waits.items() if w is not None and w[0].passes(w[1])]
        if done < len(queue):
            ready.append("run")
        if not ready:
            return all(w is None for w in waits.values())
        k = rng.choices(ready, [speed[x] for x in ready])[0]
        if k == "run":
            if queue[done][0] == "commit":
                queue[done][1].phase += 1
            done += 1
        else:
            waits[k] = next(actors[k], None)
            if waits[k] is None and k != "issue":
                left = [q for q in queue[done:] if q[0] != "commit"]
                if left or waits["issue"] is not None:
                    return False


@pytest.mark.parametrize("SB,MT", [(1, 2), (2, 1)])
def test_softmax_leaves_after_the_last_product(SB, MT):
    rng = random.Random(SB)
    assert all(_run(SB, MT, rng.randint(1, 7), True, rng) for _ in range(4000))


def test_the_last_wait_alone_is_not_enough_with_two_score_buffers():
    rng = random.Random(3)
    assert not all(_run(2, 1, rng.randint(2, 7), False, rng) for _ in range(4000))
