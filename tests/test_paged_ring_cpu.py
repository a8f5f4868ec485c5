"""The order in which the roles of the chunk kernel (csrc/paged_chunk.cu) wait for one another, restated on the host.

Every role is a generator that yields what it waits for; barriers are counters with the parity rule of an mbarrier. Roles
run in random order until all are done or none can move. What is looked for: items without blocks of keys, in any number,
must not lock the ring through which the items are handed out.
"""
import random

import pytest

SLOTS = 4  # kItemSlots


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phases = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phases = self.count, self.phases + 1

    def passed(self, parity):  # the phase of that parity is over
        return self.phases & 1 != parity


class Cta:
    """One CTA's walk over `items`, each (steps, blocks of half A, blocks of half B). `through`: the cursor of the scores looks
    through any number of items without blocks, instead of stopping behind the last item taken."""

    def __init__(self, items, stages, beside, masked, through=False):
        self.items, self.stages, self.beside, self.masked, self.through = items, stages, beside, masked, through
        many = lambda n, count: [Barrier(count) for _ in range(n)]  # noqa: E731
        self.item_full, self.item_empty = many(SLOTS, 1), many(SLOTS, 6)
        self.slot = [None] * SLOTS
        self.q_full, self.q_empty = Barrier(1), Barrier(2)
        self.k_full, self.v_full, self.k_empty, self.v_empty = many(stages, 1), many(stages, 1), many(stages, 2), many(stages, 2)
        self.s_full, self.s_free, self.p_full, self.pv_done = many(2, 1), many(2, 1), many(2, 1), many(2, 1)
        self.products = [0, 0]
        self.written = [0, 0]

    def read(self, count, release):
        yield self.item_full[count % SLOTS], (count // SLOTS) & 1
        item = self.slot[count % SLOTS]
        assert item[0] == count, "the slot holds another item"
        if release:
            self.item_empty[count % SLOTS].arrive()
        return item[1]

    def finder(self):
        for i, item in enumerate([*self.items, None]):
            yield self.item_empty[i % SLOTS], ((i // SLOTS) & 1) ^ 1
            self.slot[i % SLOTS] = (i, item)
            self.item_full[i % SLOTS].arrive()
        yield self.item_empty[i % SLOTS], (i // SLOTS) & 1  # until every reader knows that there are no more

    def queries(self):
        taken = n = 0
        while (item := (yield from self.read(taken, True))) is not None:
            taken += 1
            if item[0]:
                yield self.q_empty, (n & 1) ^ 1
                n += 1
                self.q_full.arrive()

    def keys(self):
        taken = g = 0
        while (item := (yield from self.read(taken, True))) is not None:
            taken += 1
            for _ in range(item[0]):
                for full, empty in ((self.k_full, self.k_empty), (self.v_full, self.v_empty)):
                    yield empty[g % self.stages], ((g // self.stages) & 1) ^ 1
                    full[g % self.stages].arrive()
                g += 1

    def softmax(self, h):
        taken = g = n = 0
        while (item := (yield from self.read(taken, True))) is not None:
            taken += 1
            for j in range(item[0]):
                if j < item[1 + h]:
                    yield self.s_full[h], n & 1
                    if n > 0:
                        yield self.pv_done[h], (n - 1) & 1
                    if self.beside:
                        self.s_free[h].arrive()
                    if self.masked:  # values that some rows must not see are looked over
                        yield self.v_full[g % self.stages], (g // self.stages) & 1
                    self.p_full[h].arrive()
                    n += 1
                g += 1
            if item[1 + h]:
                yield self.pv_done[h], (n - 1) & 1
            self.written[h] += 1

    def products_of(self, h):
        st = dict(taken=0, s_taken=0, s_item=None, s_more=False, s_j=0, s_g=0, s_n=0, s_items=0, end=False)
        g = n = 0

        def seek():
            while not st["s_more"] and not st["end"] and (self.through or st["s_taken"] <= st["taken"]):
                st["s_item"] = yield from self.read(st["s_taken"], False)
                st["s_taken"] += 1
                st["end"] = st["s_item"] is None
                st["s_more"] = not st["end"] and st["s_item"][0] > 0

        def scores_to(limit):
            while st["s_g"] < limit:
                yield from seek()
                if not st["s_more"]:
                    return
                if st["s_j"] == 0:
                    yield self.q_full, st["s_items"] & 1
                at = st["s_g"] % self.stages
                yield self.k_full[at], (st["s_g"] // self.stages) & 1
                if st["s_j"] < st["s_item"][1 + h]:
                    if self.beside:
                        yield self.s_free[h], (st["s_n"] & 1) ^ 1
                    elif n > 0:
                        yield self.pv_done[h], (n - 1) & 1
                    self.s_full[h].arrive()
                    st["s_n"] += 1
                self.k_empty[at].arrive()
                st["s_g"] += 1
                st["s_j"] += 1
                if st["s_j"] == st["s_item"][0]:
                    self.q_empty.arrive()
                    st["s_items"] += 1
                    st["s_j"], st["s_more"] = 0, False
                    if self.through:
                        yield from seek()

        if self.through:
            yield from scores_to(1)
        while True:
            yield from seek()
            item = yield from self.read(st["taken"], True)
            if item is None:
                return
            st["taken"] += 1
            for j in range(item[0]):
                yield from scores_to(g + (2 if self.beside else 1))
                assert st["s_g"] > g, "a product without scores"
                at = g % self.stages
                if j < item[1 + h]:
                    yield self.p_full[h], n & 1
                yield self.v_full[at], (g // self.stages) & 1
                if j < item[1 + h]:
                    self.pv_done[h].arrive()
                    n += 1
                    self.products[h] += 1
                self.v_empty[at].arrive()
                if not self.beside:
                    yield from scores_to(g + 2)
                g += 1

    def run(self, rng):
        """True if every role came to its end."""
        finder = self.finder()
        roles = [finder, self.queries(), self.keys(), self.softmax(0), self.softmax(1), self.products_of(0), self.products_of(1)]
        at = {r: None for r in roles}
        while at:
            moved = False
            for r in rng.sample(list(at), len(at)):
                want = at[r]
                if want is None or want[0].passed(want[1]):
                    moved = True
                    try:
                        at[r] = next(r)
                    except StopIteration:
                        del at[r]
            if not moved:
                assert finder in at, "nobody sees that nothing moves"
                return False
        return True


def item(rng, none):
    if rng.random() < none:
        return (0, 0, 0)
    steps = rng.choice([1, 1, 2, 3, 7])
    if rng.random() < 0.3:
        return (steps, steps, 0)  # at most 128 rows
    return (steps, rng.randint(0, steps), steps)


@pytest.mark.parametrize("stages,beside", [(3, True), (2, True), (2, False), (1, False)])
@pytest.mark.parametrize("masked", [False, True])
def test_every_order_of_items_comes_to_its_end(stages, beside, masked):
    for seed in range(60):
        rng = random.Random(seed)
        none = rng.choice([0.0, 0.2, 0.5, 0.9, 1.0])
        items = [item(rng, none) for _ in range(rng.randint(0, 30))]
        if seed % 2:  # as the kernel lists them: those with most keys first
            items.sort(key=lambda i: -i[0])
        cta = Cta(items, stages, beside, masked)
        assert cta.run(rng), items
        assert cta.products == [sum(i[1] for i in items), sum(i[2] for i in items)] and cta.written == [len(items)] * 2


def test_the_restatement_sees_a_cursor_that_looks_too_far():
    """Three items without blocks lock it where it runs an item ahead, four anywhere."""
    for before in ([], [(3, 3, 0)], [(2, 1, 2), (1, 1, 1)]):
        for empty in range(9):
            for beside in (True, False):
                items = before + [(0, 0, 0)] * empty
                assert Cta(items, 2, beside, False).run(random.Random(1))
                if empty != 3:
                    assert Cta(items, 2, beside, False, through=True).run(random.Random(1)) == (empty < SLOTS), (before, empty)
