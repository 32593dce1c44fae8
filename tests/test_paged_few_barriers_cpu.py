"""The ring of the few-row attention kernel when waits run out, on the CPU.

A model of paged_few.cu's copy warp and compute warps under random schedules (paged_chunk.cu's copy warps end alike).  A wait whose phase is not there may run
out at any time; after the first one that did, others do soon (the status bit is sticky).  A compute warp notes it for the whole
CTA and goes on; the copy warp stops.  Whatever runs out: nobody is stuck, no stage is filled again before its last copy
has landed, a part is stored by all warps or by none, only what was read from landed tiles is stored, and the CTA does
not end with a copy on its way.
"""
import random

import pytest

from test_paged_barriers_cpu import Bar


def run(seed, settle="always", check_full=True):
    r = random.Random(seed)
    stages, warps = r.choice([(3, 4), (6, 8)])
    parts = [r.randint(1, 8) for _ in range(r.randint(1, 5))]
    full, empty = [Bar(1) for _ in range(stages)], [Bar(warps) for _ in range(stages)]
    stage, flight, stored = [None] * stages, [], [0] * len(parts)
    joins, ends = [[] for _ in parts], [[] for _ in parts]  # a part's named barriers, before and after its stores
    noted = []                   # the CTA's flag
    timeouts = r.random() < .8

    def copy():
        t, ok = 0, True
        for n in parts:
            for _ in range(n):
                s = t % stages
                if t >= stages:
                    ok = not check_full or (yield full[s], t // stages - 1)
                    ok = ok and (yield empty[s], t // stages - 1)
                if not ok:
                    break
                full[s].arrive(1)

                def landed(t=t, s=s):
                    stage[s] = t
                    full[s].land(1)

                flight.append(landed)
                t += 1
            if not ok:
                break
        for c in range(max(0, t - stages), t) if settle == "always" or settle == "own" and not ok else ():
            yield full[c % stages], c // stages, "until it is there"

    def compute():
        t = 0
        for p, n in enumerate(parts):
            right = True
            for _ in range(n):
                s = t % stages
                if not (yield full[s], t // stages):
                    noted.append(True)
                right = right and stage[s] == t
                empty[s].arrive()
                t += 1
            joins[p].append(right)
            yield joins[p]
            if not noted:
                assert all(joins[p])
                stored[p] += 1
            ends[p].append(None)
            yield ends[p]

    roles = [copy()] + [compute() for _ in range(warps)]
    waits = [next(g, None) for g in roles]
    speed = [r.choice([1, 1, 5, 30]) for _ in roles]
    land, give_up, out = r.choice([1, 5, 30]), r.choice([.003, .03, .3]), False
    while any(waits):
        can, weight = [], []
        for i, w in enumerate(waits):
            if w is None:
                continue
            there = len(w) == warps if isinstance(w, list) else w[0].passes(w[1])
            if there or (timeouts and isinstance(w, tuple) and len(w) == 2):
                can.append(i)
                weight.append(speed[i] if there else speed[i] * (1 if out else give_up))
        can += ["land"] * bool(flight)
        weight += [land] * bool(flight)
        assert can, f"stuck: {seed}"
        a = r.choices(can, weight)[0]
        if a == "land":
            flight.pop(r.randrange(len(flight)))()
            continue
        w = waits[a]
        there = isinstance(w, list) or w[0].passes(w[1])
        if there and not out and not isinstance(w, list):
            assert w[0].phase == w[1] + 1, f"a wait passed for another phase: {seed}"
        out |= not there
        try:
            waits[a] = roles[a].send(there)
        except StopIteration:
            waits[a] = None
    assert not flight, f"the CTA ended with a copy on its way: {seed}"
    assert all(n in (0, warps) for n in stored)
    assert out or stored == [warps] * len(parts)


@pytest.mark.parametrize("block", range(4))
def test_waits_that_run_out(block):
    for seed in range(400 * block, 400 * (block + 1)):
        run(seed)


@pytest.mark.parametrize("form", [dict(settle="never"), dict(settle="own"), dict(check_full=False)])
def test_the_model_finds(form):
    """Copies that nobody waits for (a copy warp that leaves them alone, or waits only where a wait of its own ran out), and
    stages filled again before their last copy has landed."""
    failed = 0
    for seed in range(1600):
        try:
            run(seed, **form)
        except AssertionError:
            failed += 1
    assert failed
