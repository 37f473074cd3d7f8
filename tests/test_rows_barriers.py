"""CPU: the order of the attention kernel's waits and arrivals (csrc/row_attention.cu), as a model run in random schedules.

A wait names a barrier and the parity of the completion that it is for.  It goes through where the barrier's count of
completions has another parity than a barrier that is short of it by one: so it goes through too early where the
barrier is two completions short, which no run on a device shows for certain.  The model's roles do the kernel's waits and
arrivals in the kernel's order; every wait also knows how many completions there must have been, and a wait that goes
through with fewer, or a state that nothing leaves, fails.
"""

from __future__ import annotations

import random

import pytest

SLOTS = 4  # ring slots: K in 0 and 2, V in 1 and 3


class Bar:
    def __init__(self, name, arrivals=1):
        self.name, self.arrivals, self.pending, self.done = name, arrivals, arrivals, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.done = self.arrivals, self.done + 1


class Item:
    """Half blocks of both row tiles, first block with keys that some row does not see, and whether there is such a key."""

    def __init__(self, halves, washed, hidden):
        self.halves, self.washed, self.hidden = halves, washed, hidden
        self.blocks = (max(halves) + 1) // 2

    def reads(self, tile):  # the tile looks at what the washing noted
        return self.hidden and self.halves[tile] > 2 * self.washed


class Model:
    """mode: "halves" (head_dim 128), "ahead" (64: a half's scores are loaded while the other is worked on), "e4m3"."""

    def __init__(self, items, mode, early_wait=True):
        self.items, self.e4m3, self.ahead, self.early_wait = items, mode == "e4m3", mode == "ahead", early_wait
        self.raw_full, self.raw_empty = Bar("raw_full"), Bar("raw_empty", 4)
        self.full = [Bar(f"full {s}", 4 if self.e4m3 and s & 1 else 1) for s in range(SLOTS)]
        self.empty = [Bar(f"empty {s}", 2) for s in range(SLOTS)]
        self.q_full, self.q_empty = Bar("q_full"), Bar("q_empty", 2)
        self.s_full = [[Bar(f"s_full {t} {h}") for h in range(2)] for t in range(2)]
        self.p_full = [[Bar(f"p_full {t} {h}", 4) for h in range(2)] for t in range(2)]
        self.o_full = [Bar(f"o_full {t}") for t in range(2)]
        self.v_clean = [Bar(f"v_clean {s}", 4) for s in range(2)]
        self.bad_read = [[Bar(f"bad_read {t} {i}", 4) for i in range(2)] for t in range(2)]
        # what completes by itself, each queue in order: copies, and the products of either tile
        self.copies, self.products = [], ([], [])
        self.roles = {"loads": self.loads(), "queries": self.queries(), "mma 0": self.mma(0), "mma 1": self.mma(1)}
        for t in range(2):
            for w in range(4):
                self.roles[f"softmax {t} {w}"] = self.softmax(t)
        if self.e4m3:
            for w in range(4):
                self.roles[f"widen {w}"] = self.widen()

    # A role yields (barrier, completions that there must have been).
    def loads(self):
        n = 0
        for it in self.items:
            for _ in range(it.blocks):
                for v in range(2):
                    s, turn = n % SLOTS, n // SLOTS
                    if self.e4m3 and v:
                        if n // 2:
                            yield self.raw_empty, n // 2
                        self.copies.append(self.raw_full)
                    else:
                        if turn:
                            yield self.empty[s], turn
                        self.copies.append(self.full[s])
                    n += 1

    def queries(self):
        for i in range(len(self.items)):
            if i:
                yield self.q_empty, i
            self.copies.append(self.q_full)

    def mma(self, t):
        slot, used, p_done, cleaned, todo = 0, [0] * SLOTS, [0, 0], [0, 0], self.products[t]

        def landed(s):
            used[s] += 1
            return self.full[s], used[s]

        for i, it in enumerate(self.items):
            halves, blocks = it.halves[t], it.blocks
            yield self.q_full, i + 1
            yield landed(slot)
            todo.extend(self.s_full[t][h] for h in range(min(halves, 2)))
            if blocks == 1:
                todo.append(self.q_empty)
            todo.append(self.empty[slot])
            slot = (slot + 1) % SLOTS
            for j in range(blocks):
                v, slot, last = slot, (slot + 1) % SLOTS, j == blocks - 1
                yield landed(v)
                if not last:
                    yield landed(slot)
                if j >= it.washed and not self.e4m3:
                    cleaned[v >> 1] += 1
                    yield self.v_clean[v >> 1], cleaned[v >> 1]
                for h in range(2):
                    k = 2 * j + h
                    if k < halves:
                        p_done[h] += 1
                        yield self.p_full[t][h], p_done[h]
                        if k == halves - 1:
                            todo.append(self.o_full[t])
                        if k + 2 < halves:
                            todo.append(self.s_full[t][h])
                todo.append(self.empty[v])
                if not last:
                    todo.append(self.empty[slot])
                    if j + 2 == blocks:
                        todo.append(self.q_empty)
                    slot = (slot + 1) % SLOTS

    def softmax(self, t):
        scores, outs, block, noted, idle = [0, 0], 0, 0, [0, 0], False
        for it in self.items:
            halves, other = it.halves[t], it.halves[t ^ 1]
            block0, block = block, block + it.blocks
            mine, theirs = noted[t], noted[t ^ 1]
            noted[t] += it.reads(t)
            noted[t ^ 1] += it.reads(t ^ 1)
            if halves == 0:
                idle = True
                continue
            was_idle, idle = idle, False
            washes = not self.e4m3 and not (halves < other or (halves == other and t == 1))
            washed = it.washed if washes else it.blocks
            if not self.ahead and washed == 0 and was_idle and self.early_wait:
                yield self.s_full[t][0], scores[0] + 1
            if self.ahead:
                scores[0] += 1
                yield self.s_full[t][0], scores[0]
            for k in range(halves):
                h, j = k & 1, k // 2
                if h == 0 and j >= washed:
                    if j == it.washed and it.reads(t ^ 1) and theirs >= 2:
                        yield self.bad_read[t ^ 1][theirs & 1], theirs // 2
                    b = block0 + j
                    yield self.full[(b & 1) * 2 + 1], b // 2 + 1
                    self.v_clean[b & 1].arrive()
                if not self.ahead:
                    scores[h] += 1
                    yield self.s_full[t][h], scores[h]
                    if self.e4m3 and h == 0:
                        b = block0 + j
                        yield self.full[(b & 1) * 2 + 1], b // 2 + 1
                elif k + 1 < halves:
                    scores[1 - h] += 1
                    yield self.s_full[t][1 - h], scores[1 - h]
                self.p_full[t][h].arrive()
            outs += 1
            yield self.o_full[t], outs
            if it.reads(t):
                self.bad_read[t][mine & 1].arrive()

    def widen(self):
        n, noted = 1, [0, 0]
        for it in self.items:
            for t in range(2):
                if it.reads(t) and noted[t] >= 2:
                    yield self.bad_read[t][noted[t] & 1], noted[t] // 2
            for _ in range(it.blocks):
                s = n % SLOTS
                yield self.raw_full, n // 2 + 1
                if n >= SLOTS:
                    yield self.empty[s], n // SLOTS
                self.full[s].arrive()
                self.raw_empty.arrive()
                n += 2
            for t in range(2):
                noted[t] += it.reads(t)

    def run(self, rng):
        """None, or what went wrong.  Roles and queues have speeds of their own, some far apart."""
        waits = {}

        def go_on(name):
            try:
                waits[name] = next(self.roles[name])
            except StopIteration:
                waits.pop(name, None)

        for name in self.roles:
            go_on(name)
        speed = {name: rng.choice([1, 1, 1, 5, 20]) for name in [*self.roles, "copies", "products 0", "products 1"]}
        queues = {"copies": self.copies, "products 0": self.products[0], "products 1": self.products[1]}
        while waits:
            # through: not in the phase that is waited for (parity alone says so)
            ready = [name for name, (bar, n) in waits.items() if (bar.done & 1) != ((n - 1) & 1)]
            ready += [name for name, queue in queues.items() if queue]
            if not ready:
                return "nothing goes on: " + ", ".join(f"{name} at {bar.name} {bar.done} of {n}"
                                                       for name, (bar, n) in waits.items())
            name = rng.choices(ready, [speed[r] for r in ready])[0]
            if name in queues:
                queues[name].pop(0).arrive()
                continue
            bar, n = waits[name]
            if bar.done < n:
                return f"{name} passes {bar.name} after {bar.done} of {n}"
            go_on(name)
        return None


def _items(rng):
    """Items as plans make them: one tile or two, a second one that ends earlier or starts later, pieces of units."""
    items = []
    for _ in range(rng.randint(3, 14)):
        blocks = rng.choice([1, 1, 1, 2, 3])
        n = 2 * blocks - rng.randint(0, 1)
        halves = {"one": (n, 0), "both": (n, n), "longer": (max(n - rng.choice([1, 2]), 0), n),
                  "second": (0, min(n, 2))}[rng.choice(["one", "both", "longer", "second"])]
        blocks = (max(halves) + 1) // 2
        hidden = rng.random() < 0.7
        items.append(Item(halves, rng.randint(max(0, blocks - 3), blocks - 1) if hidden else rng.choice([blocks - 1, blocks]),
                          hidden))
    return items


@pytest.mark.parametrize("mode", ["halves", "ahead", "e4m3"])
def test_no_wait_goes_through_early_and_none_is_left(mode):
    for seed in range(400):
        rng = random.Random(seed)
        assert Model(_items(rng), mode).run(rng) is None, seed


def test_the_model_sees_a_missing_wait():
    """Without the wait for an item's first scores that a tile without work in the item before does, washing warps run so
    far ahead that a slot's phases can no longer be told apart."""
    found = set()
    for seed in range(3000):
        rng = random.Random(seed)
        wrong = Model(_items(rng), "halves", early_wait=False).run(rng)
        if wrong:
            found.add(wrong.split(" after")[0].rsplit(" ", 1)[0])
    assert any("passes full" in w or "passes bad_read" in w or "passes v_clean" in w for w in found), found
