"""Every order in which the warps of the MXFP4 products (csrc/mxfp4_stream.cu, mxfp4_tiles.cu) can reach their barriers, on a model.  A wait on an mbarrier
names a phase by its parity alone, so it is right only while nobody is two phases behind; copies and products are asynchronous."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llmopt_b200", "csrc")


class Model:
    """``programs``: per warp a list of steps (barrier, phase, effects) -- a wait (barrier None: none) and what follows it at once.  Effects:
    ("arrive", barrier), ("copy", barrier, which), ("product", barriers): a copy or product is under way until some later point, products
    end in the order of their issue, and then arrive.  ``needs``: arrivals and landed copies that a phase of a barrier takes."""

    def __init__(self, programs, needs):
        self.programs, self.needs = [list(program) for program in programs], needs
        self.start = ((0,) * len(self.programs), (), frozenset(), ())

    def arrive(self, counts, barrier):
        counts = dict(counts)
        over, had = counts.get(barrier, (0, 0))
        had += 1
        counts[barrier] = (over + 1, 0) if had == self.needs[barrier] else (over, had)
        return tuple(sorted(counts.items()))

    def events(self, state):
        """What ends without a warp: copies that land, the oldest product."""
        places, counts, copies, products = state
        for copy in copies:
            yield places, self.arrive(counts, copy[0]), copies - {copy}, products
        if products:
            after = counts
            for barrier in products[0]:
                after = self.arrive(after, barrier)
            yield places, after, copies, products[1:]

    def effects(self, state, warp, effects):
        places, counts, copies, products = state
        places = places[:warp] + (places[warp] + 1,) + places[warp + 1:]
        for effect in effects:
            if effect[0] == "arrive":
                counts = self.arrive(counts, effect[1])
            elif effect[0] == "copy":
                copies = copies | {effect[1:]}
            else:
                products = products + (effect[1],)
        return places, counts, copies, products

    def passes(self, state, barrier, phase):
        """(whether a wait for the phase ends, whether it should)."""
        over = dict(state[1]).get(barrier, (0, 0))[0]
        return barrier is None or (over - 1) % 2 == phase % 2, barrier is None or over > phase

    def orders(self):
        """What can go wrong, over all orders: waits that end too early ("early"), warps that wait for good ("stuck")."""
        wrong, seen, pending = set(), set(), [self.start]
        while pending:
            state = pending.pop()
            if state in seen:
                continue
            seen.add(state)
            following = list(self.events(state))
            for warp, program in enumerate(self.programs):
                if state[0][warp] == len(program):
                    continue
                barrier, phase, effects = program[state[0][warp]]
                ends, over = self.passes(state, barrier, phase)
                if ends and not over:
                    wrong.add("early")
                elif ends:
                    following.append(self.effects(state, warp, effects))
            if not following and any(place < len(program) for place, program in zip(state[0], self.programs)):
                wrong.add("stuck")
            pending.extend(following)
        return wrong


    def ways_out(self, leave):
        """The same where any wait can run out: its warp ends there (place p becomes ~p).  States whose warps all have ended, some by
        giving up, are handed to ``leave``, which says what can go wrong from there on."""
        wrong, seen, pending = set(), set(), [self.start]
        while pending:
            state = pending.pop()
            if state in seen:
                continue
            seen.add(state)
            pending.extend(self.events(state))
            places, ended = state[0], True
            for warp, program in enumerate(self.programs):
                place = places[warp]
                if place == len(program) or place < 0:
                    continue
                ended = False
                barrier, phase, effects = program[place]
                ends, over = self.passes(state, barrier, phase)
                if ends and not over:
                    wrong.add("early")
                elif ends:
                    pending.append(self.effects(state, warp, effects))
                if barrier is not None:
                    pending.append((places[:warp] + (~place,) + places[warp + 1:], *state[1:]))
            if ended and min(places) < 0:
                wrong |= leave(state)
        return wrong


def waits_for(model, state, waits, drained):
    """Whether something is still under way when all of ``waits``, and that for the products issued (``drained``), have ended, or one of
    them never does."""
    wrong, pending, seen = set(), [state], set()
    while pending:
        state = pending.pop()
        if state in seen:
            continue
        seen.add(state)
        following = list(model.events(state))
        if all(model.passes(state, *wait)[0] for wait in waits) and not (drained and state[3]):
            if state[2] or state[3]:
                wrong.add("left")
            continue
        if not following:
            wrong.add("stuck")
        pending.extend(following)
    return wrong


def started(model, state, warp):
    """Stages whose copies a warp has started."""
    program, place = model.programs[warp], state[0][warp]
    place = place if place >= 0 else ~place
    return sum(effect[0] == "copy" for step in program[:place] for effect in step[2])


def stream(depth, ring):
    """The warps of a CTA of mxfp4_stream.cu: copies (of the first stages without a wait), exponents, products, read-out."""
    stages = range(depth)
    needs = {("sums",): 1, **{(name, s): need for name, need in (("full", 2), ("scales", 1), ("empty", 1)) for s in range(ring)}}
    copies = [(("empty", i % ring) if i >= ring else None, i // ring - 1, [("arrive", ("full", i % ring)), ("copy", ("full", i % ring), i)]) for i in stages]
    exponents = [(("empty", i % ring), i // ring - 1, [("arrive", ("scales", i % ring))]) for i in stages]
    products = [step for i in stages for step in (
        (("full", i % ring), i // ring, []),
        (("scales", i % ring), i // ring, [("product", (("empty", i % ring),) + ((("sums",),) if i + 1 == depth else ()))]))]
    return Model([copies, exponents, products, [(("sums",), 0, [])]], needs)


@pytest.mark.parametrize("depth,ring", [(1, 1), (1, 2), (2, 2), (3, 2), (5, 2), (4, 3)])
def test_streams_wait_for_no_phase_too_early_and_for_none_for_good(depth, ring):
    assert stream(depth, ring).orders() == set()


@pytest.mark.parametrize("depth,ring", [(1, 1), (1, 2), (2, 2), (3, 2), (4, 2), (4, 3)])
@pytest.mark.parametrize("awaited", [True, False])
def test_nothing_is_under_way_when_a_stream_has_given_up(depth, ring, awaited):
    """The copies that the ring can still hold, and the products, are awaited when all warps have ended.  The model sees what is left where the
    warps that copy and multiply wait at their own end, and only if they know of a failure by then: another may give up after it."""
    model = stream(depth, ring)

    def leave(state):
        stages = started(model, state, 0)
        waits = [(("full", i % ring), i // ring) for i in range(max(0, stages - ring), stages)]
        return waits_for(model, state, waits if awaited or state[0][0] < 0 else [], awaited or state[0][2] < 0)

    assert model.ways_out(leave) == (set() if awaited else {"left"})


def pair(tiles, depth, ring, relayed=True):
    """The warps of a pair of CTAs (one of those that do the same), over ``tiles`` of ``depth`` stages.  Not relayed: the warps that bring
    exponents do not wait until a stage is empty."""
    stages = range(tiles * depth)
    needs = {}
    for s in range(ring):
        # of the first CTA's copies its own arrival and both halves
        needs.update({("full", s): 3, ("scales", s): 2, ("laid", s): 1, ("empty", 0, s): 1, ("empty", 1, s): 1, ("vacant", 0, s): 1, ("vacant", 1, s): 1})
    for b in range(2):
        needs.update({("sums_full", 0, b): 1, ("sums_full", 1, b): 1, ("sums_empty", b): 2})
    programs = []
    for rank in (0, 1):
        post = (("arrive", "full"),) if rank == 0 else ()
        programs.append([(("empty", rank, i % ring), i // ring - 1,
                          [("arrive", ("vacant", rank, i % ring))] + [("arrive", ("full", i % ring)) for _ in post] + [("copy", ("full", i % ring), rank, i)])
                         for i in stages])
        programs.append([(("vacant", rank, i % ring) if relayed else None, i // ring,
                          [("arrive", ("scales" if rank == 0 else "laid", i % ring))]) for i in stages])
        programs.append([(("sums_full", rank, t % 2), t // 2, [("arrive", ("sums_empty", t % 2))]) for t in range(tiles)])
    programs.append([(("laid", i % ring), i // ring, [("arrive", ("scales", i % ring))]) for i in stages])
    issuer = []
    for i in stages:
        if i % depth == 0:
            issuer.append((("sums_empty", i // depth % 2), i // depth // 2 - 1, []))
        issuer.append((("full", i % ring), i // ring, []))
        done = [("empty", 0, i % ring), ("empty", 1, i % ring)]
        if i % depth == depth - 1:
            done += [("sums_full", 0, i // depth % 2), ("sums_full", 1, i // depth % 2)]
        issuer.append((("scales", i % ring), i // ring, [("product", tuple(done))]))
    return Model(programs + [issuer], needs)


@pytest.mark.parametrize("tiles,depth,ring", [(1, 1, 2), (1, 3, 2), (2, 2, 2), (3, 1, 2), (2, 1, 1)])
def test_pairs_wait_for_no_phase_too_early_and_for_none_for_good(tiles, depth, ring):
    assert pair(tiles, depth, ring).orders() == set()


@pytest.mark.parametrize("tiles,depth,ring", [(1, 1, 2), (1, 2, 1), (1, 2, 2), (2, 1, 2)])
@pytest.mark.parametrize("awaited", [True, False])
def test_nothing_is_under_way_when_a_pair_has_given_up(tiles, depth, ring, awaited):
    """The first CTA waits for the copies of both, and makes up for what a stage lacks that one of them alone came to ask for.  The model sees
    what is left or waited for in vain where the warps that copy and multiply wait at their own end, only if they know of a failure by
    then, and for the stages that the first CTA asked for."""
    model = pair(tiles, depth, ring)

    def leave(state):
        first, second = started(model, state, 0), started(model, state, 3)
        places, counts, copies, products = state
        if not awaited:
            waits = [(("full", i % ring), i // ring) for i in range(max(0, first - ring), first)]
            return waits_for(model, state, waits if places[0] < 0 else [], places[-1] < 0)
        last = max(first, second)
        for i in range(max(0, last - ring), last):
            if i >= first:  # its own word, and its half of the bytes, which it does not count
                counts = model.arrive(model.arrive(counts, ("full", i % ring)), ("full", i % ring))
            if i >= second:
                counts = model.arrive(counts, ("full", i % ring))
        waits = [(("full", i % ring), i // ring) for i in range(max(0, last - ring), last)]
        return waits_for(model, (places, counts, copies, products), waits, True)

    wrong = model.ways_out(leave)
    assert wrong == set() if awaited else wrong & {"left", "stuck"}


def test_the_model_sees_exponents_that_do_not_wait():
    assert pair(1, 3, 2, relayed=False).orders() & {"early", "stuck"}


def test_what_crosses_a_pair_is_of_the_clusters_scope():
    """An arrival or wait that names no scope is of the CTA's and orders nothing between threads of two CTAs."""
    with open(os.path.join(CSRC, "mxfp4_tiles.cu")) as file:
        source = file.read()
    arrivals = re.findall(r"mbarrier\.arrive\S*", source)
    assert arrivals and all(".cluster.shared::cluster" in arrival for arrival in arrivals)
    wait = re.findall(r"mbarrier\.try_wait\S*", source)
    assert wait and all(".cluster.shared::cta" in form for form in wait)
    # waits of the CTA's scope are those for what only this CTA's threads say
    assert set(re.findall(r"warp_wait\((\w+)", source)) == {"laid", "vacant"}
