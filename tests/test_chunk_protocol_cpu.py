"""The barrier protocol of the attention of several new tokens as a model that runs on the CPU under random schedules.

The kernel's warps (metile_b200/csrc/paged_chunk.cuh) hand units, tiles of keys and values, scores and weights to one another
through mbarriers, whose waits see only the parity of a phase.  The model has the same roles, waits and arrivals in the same
order; copies land and the tensor cores work at arbitrary times.  What is read before it is there, overwritten before it has been
read, or waited for in vain is a fault.  The number of slots of the ring comes from the kernel's header."""

import pathlib
import random
import re
from collections import defaultdict

import pytest

from tests.helpers import host_program


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1


class Fault(Exception):
    pass


def expect(found, wanted, *what):
    if found != wanted:
        raise Fault(f"{what}: found {found}, expected {wanted}")


class Model:
    """units: (steps of 64 tokens, query tiles at work, first token tile whose values are looked at) each."""

    def __init__(self, units, slots, per_tile, groups, rng, spoil=None):
        self.units, self.slots, self.per_tile, self.groups, self.rng, self.spoil = units, slots, per_tile, groups, rng, spoil
        self.bars = {"q_full": Barrier(1), "q_empty": Barrier(2 * groups + 1), "to_fix": Barrier(1 if spoil == "to_fix" else groups), "fixed": Barrier(1)}
        for slot in range(slots):
            self.bars["full", slot], self.bars["empty", slot] = Barrier(1), Barrier(groups)
        for g in range(groups):
            self.bars["turn", g] = Barrier(1)
            for place in range(2):
                for name in "spo":
                    self.bars[name, g, place] = Barrier(1)
        self.unit = self.count = None
        self.ring, self.mended, self.scores, self.results = [None] * slots, defaultdict(bool), {}, {}
        self.queues = [[] for _ in range(groups)]

    def wait(self, name, parity, phase):
        """Until the parity says so; that must be when `phase` has completed."""
        bar = self.bars[name]
        while (bar.phase & 1) == parity:
            yield
        if bar.phase <= phase:
            raise Fault(f"{name} passed ahead of phase {phase}")

    def tiles(self, unit):
        return -(-unit[0] // self.per_tile)

    def loader(self):
        item = 0

        def load(count, tile, values):
            nonlocal item
            slot, turn = item % self.slots, item // self.slots
            if turn:
                yield from self.wait(("empty", slot), (turn - 1) & 1, turn - 1)
            yield
            self.ring[slot] = (count, tile, values)
            self.bars["full", slot].arrive()
            item += 1

        for count, unit in enumerate(self.units + [None]):
            tiles = self.tiles(unit) if unit else 0
            if tiles:
                yield from load(count, 0, 0)
                yield from load(count, 0, 1)
            if count:
                yield from self.wait("q_empty", (count - 1) & 1, count - 1)
            self.unit, self.count = unit, count
            self.bars["q_full"].arrive()
            yield
            for tile in range(1, tiles):
                yield from load(count, tile, 0)
                yield from load(count, tile, 1)

    def issuer(self, g):
        queue, item, fixed, count, turns = self.queues[g], 0, 0, 0, 0
        parity, phases = [0, 0], [0, 0]
        while True:
            yield from self.wait("q_full", count & 1, count)
            expect(self.count, count, "unit")
            unit = self.unit
            if unit is None:
                return
            steps, active, fix_from = unit
            works, tiles = g < active, self.tiles(unit)
            if steps == 0:
                self.bars["q_empty"].arrive()
                count += 1
                continue

            def arrived(it):
                yield from self.wait(("full", it % self.slots), it // self.slots & 1, it // self.slots)
                expect(self.ring[it % self.slots], (count, (it - item) // 2, (it - item) % 2), "tile")

            def scores(step):
                it = item + 2 * (step // self.per_tile)
                if works:
                    queue.append(("scores", count, g, step, it % self.slots))
                    queue.append(("commit", ("s", g, step & 1)))
                if step % self.per_tile == self.per_tile - 1 or step == steps - 1:
                    queue.append(("commit", ("empty", it % self.slots)))
                if step == steps - 1:
                    queue.append(("commit", "q_empty"))

            for step in range(min(2, steps)):
                if step % self.per_tile == 0:
                    yield from arrived(item + 2 * (step // self.per_tile))
                scores(step)
                yield
            for step in range(steps):
                tile, value_item, ahead, place = step // self.per_tile, item + 2 * (step // self.per_tile) + 1, step + 2, step & 1
                if step % self.per_tile == 0:
                    yield from arrived(value_item)
                    if tile >= fix_from and (g == 0 or self.spoil != "to_fix"):
                        self.bars["to_fix"].arrive()
                    if ahead < steps:
                        yield from arrived(item + 2 * (ahead // self.per_tile))
                    if tile >= fix_from:
                        yield from self.wait("fixed", fixed & 1, fixed)
                        expect(self.mended[count, tile], True, "values not looked at")
                        fixed += 1
                if works:
                    yield from self.wait(("p", g, place), parity[place], phases[place])
                    parity[place] ^= 1
                    phases[place] += 1
                    if active == 2:
                        yield from self.wait(("turn", g), (turns & 1) ^ (g == 0), turns - (g == 0))
                        turns += 1
                    queue.append(("results", count, g, step, value_item % self.slots))
                    queue.append(("commit", ("o", g, place)))
                if step % self.per_tile == self.per_tile - 1 or step == steps - 1:
                    queue.append(("commit", ("empty", value_item % self.slots)))
                if ahead < steps:
                    scores(ahead)
                if active == 2:
                    self.bars["turn", 1 - g].arrive()
                yield
            item += 2 * tiles
            count += 1

    def tensor(self, g):
        queue = self.queues[g]
        while True:
            if queue:
                operation = queue.pop(0)
                if operation[0] == "commit":
                    self.bars[operation[1]].arrive()
                else:
                    kind, count, _, step, slot = operation
                    expect(self.ring[slot], (count, step // self.per_tile, int(kind == "results")), operation)
                    if kind == "scores":
                        self.scores[g, step & 1] = ("scores", count, step)
                    else:
                        expect(self.scores.get((g, step & 1)), ("weights", count, step), operation)
                        self.results[g] = (count, step)
                for _ in range(self.rng.randrange(3)):
                    yield
            yield

    def fixer(self):
        fixed = count = 0
        while True:
            yield from self.wait("q_full", count & 1, count)
            expect(self.count, count, "unit")
            unit = self.unit
            self.bars["q_empty"].arrive()
            if unit is None:
                return
            for tile in range(unit[2], self.tiles(unit)):
                yield from self.wait("to_fix", fixed & 1, fixed)
                fixed += 1
                self.mended[count, tile] = True
                self.bars["fixed"].arrive()
                yield
            count += 1

    def rows(self, g):
        count, parity, seen = 0, [0, 0], [0, 0]
        while True:
            yield from self.wait("q_full", count & 1, count)
            expect(self.count, count, "unit")
            unit = self.unit
            self.bars["q_empty"].arrive()
            if unit is None:
                return
            steps = unit[0] if g < unit[1] else 0
            for step in range(steps):
                place = step & 1
                yield from self.wait(("s", g, place), parity[place], seen[place])
                parity[place] ^= 1
                seen[place] += 1
                expect(self.scores.get((g, place)), ("scores", count, step), "scores")
                for _ in range(self.rng.randrange(4)):
                    yield
                if step and self.rng.random() < 0.3:  # the row's maximum moves
                    yield from self.wait(("o", g, place ^ 1), parity[place ^ 1] ^ 1, seen[place ^ 1] - 1)
                    expect(self.results.get(g), (count, step - 1), "results so far")
                self.scores[g, place] = ("weights", count, step)
                self.bars["p", g, place].arrive()
                yield
            if steps:
                place = (steps - 1) & 1
                yield from self.wait(("o", g, place), parity[place] ^ 1, seen[place] - 1)
                for _ in range(self.rng.randrange(6)):
                    expect(self.results.get(g), (count, steps - 1), "results")
                    yield
            count += 1

    def state(self):
        return tuple(bar.phase * 100 + bar.left for bar in self.bars.values()), tuple(len(q) for q in self.queues)

    def run(self):
        roles = {"loader": self.loader(), "fixer": self.fixer()}
        for g in range(self.groups):
            roles["issuer", g], roles["tensor", g], roles["rows", g] = self.issuer(g), self.tensor(g), self.rows(g)
        weight = {name: self.rng.choice((1, 1, 5, 20)) for name in roles}
        idle = 0
        while any(name[0] != "tensor" for name in roles):
            names = [name for name in roles for _ in range(weight[name])]
            before = self.state()
            name = self.rng.choice(names)
            try:
                next(roles[name])
            except StopIteration:
                del roles[name]
                idle = 0
                continue
            idle = idle + 1 if self.state() == before else 0
            if idle > 5000:
                raise Fault("nobody can go on")


def random_units(rng, per_tile, groups):
    units = []
    for _ in range(rng.randrange(1, 6)):
        steps = rng.choice((0, 1, 2, 3, 4, 5, 7, 11))
        tiles = -(-steps // per_tile)
        units.append((steps, rng.randint(1, groups), rng.randrange(tiles) if tiles else 0))
    return units


@pytest.fixture(scope="module")
def shapes(tmp_path_factory):
    """(slots, steps of a tile, query tiles) for the head dimensions 64, 128 and 256."""
    return host_program(str(tmp_path_factory.mktemp("shapes")), '#include <cstdio>\n#include "../../include/metile_b200.h"\n#include "paged_chunk.cuh"\n'
                        "template <int kD> void show() { using Shape = mt::ChunkShape<kD>; printf(\"%d %d %d\\n\", Shape::kSlots, Shape::kSteps, Shape::kGroups); }\n"
                        "int main() { show<64>(); show<128>(); show<256>(); return 0; }\n")


def test_random_schedules(shapes):
    assert len(shapes) == 3
    for seed in range(60):
        rng = random.Random(seed)
        slots, per_tile, groups = rng.choice(shapes)
        Model(random_units(rng, per_tile, groups), slots, per_tile, groups, rng).run()


def test_the_model_finds_a_wait_that_is_two_phases_behind(shapes):
    """Handing values on by one of the issuers alone lets the other be lapped."""
    found = 0
    for seed in range(60):
        rng = random.Random(seed)
        slots, per_tile, groups = shapes[1]
        try:
            Model(random_units(rng, per_tile, groups), slots, per_tile, groups, rng, spoil="to_fix").run()
        except Fault:
            found += 1
    assert found > 0


def test_tensor_memory_is_taken_before_the_next_kernel_may_start():
    """A dependent kernel's block may share an SM with one of the kernel in front.  If it could take the tensor memory first, the one in
    front would wait for it, and it for the end of the one in front: so each block lets dependents start behind a barrier behind
    its own allocation."""
    sources = pathlib.Path(__file__).resolve().parent.parent / "metile_b200" / "csrc"
    found = 0
    for source in sources.glob("*.cuh"):
        text = re.sub(r"//[^\n]*", "", source.read_text())
        for kernel in re.split(r"__global__", text)[1:]:
            if "ptx::tmem_alloc(" not in kernel:
                continue
            found += 1
            at = kernel.index("ptx::tmem_alloc("), kernel.index("griddep_launch_dependents(")
            assert at[0] < kernel.index("__syncthreads()", at[0]) < at[1], source.name
    assert found >= 2
