"""The stages of the prompt attention kernel, replayed on the CPU: who loads, multiplies and gives back which stage, with barriers
whose waits tell only neighbouring turns apart, in random orders of what may happen next.  No stage may be loaded again before
both tiles' multiplications are through with it, nothing may be multiplied before it is there, and nobody may wait for good.

The kernel's layout is read from its source: keys and values each have a ring of their own.  One ring that both share in turn is
replayed too, to show that the replay sees what goes wrong with it: with an odd number of stages the two loaders take turns on a
stage, and a loader whose turn before last is still in use takes it for given back."""
import os
import random
import re

import pytest

from tests.conftest import ROOT

KEYS, VALUES = 0, 1


class Overwritten(Exception):
    pass


class Stuck(Exception):
    pass


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):      # what a parity wait sees: the phase before the one under way has this parity
        return (self.phase & 1) != parity


class Block:
    """pieces: per pair, the position blocks of tile 0 and of tile 1 as (first, last); rings: stages of the keys and of the values,
    or (n,) for one ring that they share in turn."""

    def __init__(self, pieces, rings, rng):
        self.pieces, self.rings, self.rng = pieces, rings, rng
        n = sum(rings)
        self.full, self.empty = [Barrier(1) for _ in range(n)], [Barrier(2) for _ in range(n)]
        self.s_full, self.o_full, self.p_full = ([Barrier(1) for _ in range(2)] for _ in range(3))
        self.holds = [None] * n       # (kind, fill) whose copy has landed
        self.uses = {}                # (kind, fill): multiplications that have yet to read it
        self.tensor = []              # the tensor core's queue
        self.copies = []
        self.fills = [(p, j) for p, (a, b) in enumerate(pieces) for j in range(min(a[0], b[0]), max(a[1], b[1]))
                      if a[0] <= j < a[1] or b[0] <= j < b[1]]

    def place(self, kind, fill):
        """Stage and parity of the turn that a fill has there."""
        if len(self.rings) == 1:
            turn = 2 * fill + kind
            return turn % self.rings[0], turn // self.rings[0] & 1
        return fill % self.rings[kind] + (self.rings[KEYS] if kind else 0), fill // self.rings[kind] & 1

    def here(self, x, fill):
        p, j = self.fills[fill]
        first, last = self.pieces[p][x]
        return first <= j < last

    def loader(self, kind):
        for fill in range(len(self.fills)):
            s, ph = self.place(kind, fill)
            yield lambda: self.empty[s].passed(ph ^ 1)
            if self.holds[s] is not None and self.uses[self.holds[s]]:
                raise Overwritten((kind, fill, self.holds[s]))
            self.uses[kind, fill] = sum(self.here(x, fill) for x in range(2))
            self.holds[s] = None
            self.copies.append((s, kind, fill))

    def issuer(self, x):
        p_count, before = 0, None
        for fill, (p, j) in enumerate(self.fills):
            (ks, kph), (vs, vph) = self.place(KEYS, fill), self.place(VALUES, fill)
            if not self.here(x, fill):
                yield lambda: self.full[ks].passed(kph)
                yield lambda: self.full[vs].passed(vph)
                self.empty[ks].arrive()
                self.empty[vs].arrive()
                continue
            first, last = self.pieces[p][x]
            yield lambda: self.full[ks].passed(kph)
            if j > first:
                yield lambda: self.p_full[x].passed(p_count & 1)
                p_count += 1
                self.tensor.append((VALUES, before))
            self.tensor += [(KEYS, fill), self.s_full[x]]
            yield lambda: self.full[vs].passed(vph)
            before = fill
            if j + 1 == last:
                yield lambda: self.p_full[x].passed(p_count & 1)
                p_count += 1
                self.tensor += [(VALUES, fill), self.o_full[x]]

    def softmax(self, x):
        s_count = o_count = 0
        before = None
        for p, ranges in enumerate(self.pieces):
            first, last = ranges[x]
            for fill, (q, j) in enumerate(self.fills):
                if q != p or not self.here(x, fill):
                    continue
                yield lambda: self.s_full[x].passed(s_count & 1)
                s_count += 1
                self.empty[self.place(KEYS, fill)[0]].arrive()
                if j > first:
                    self.empty[before].arrive()
                before = self.place(VALUES, fill)[0]
                yield None
                self.p_full[x].arrive()
            if first < last:
                yield lambda: self.o_full[x].passed(o_count & 1)
                o_count += 1
                self.empty[before].arrive()

    def tensor_core(self):
        while True:
            yield lambda: self.tensor
            op = self.tensor.pop(0)
            if isinstance(op, Barrier):
                op.arrive()
                continue
            if self.holds[self.place(*op)[0]] != op:
                raise Overwritten(op)
            self.uses[op] -= 1

    def copier(self):
        while True:
            yield lambda: self.copies
            s, kind, fill = self.copies.pop(self.rng.randrange(len(self.copies)))
            if self.holds[s] is not None:
                raise Overwritten((kind, fill, self.holds[s]))
            self.holds[s] = (kind, fill)
            self.full[s].arrive()

    def run(self):
        roles = [self.loader(KEYS), self.loader(VALUES), self.issuer(0), self.issuer(1), self.softmax(0), self.softmax(1)]
        endless = [self.tensor_core(), self.copier()]
        weights = {id(r): 10.0 ** self.rng.uniform(-3, 0) for r in roles + endless}   # some of them are slow
        waits = {id(r): next(r, StopIteration) for r in roles + endless}
        alive = [r for r in roles if waits[id(r)] is not StopIteration]
        while alive:
            able = [r for r in alive + endless if waits[id(r)] is None or waits[id(r)]()]
            if not able:
                raise Stuck
            r = self.rng.choices(able, [weights[id(a)] for a in able])[0]
            waits[id(r)] = next(r, StopIteration)
            if waits[id(r)] is StopIteration:
                alive.remove(r)


def pieces(rng):
    """A few pairs: tiles whose last blocks differ, tiles that a window starts at different blocks, second tiles without rows."""
    out = []
    for _ in range(rng.randint(1, 5)):
        first, n = rng.randint(0, 3), rng.randint(1, 7)
        a = (first, first + n)
        b = rng.choice([a, (first, first + n + 1), (first + 1, first + n + 1), (0, 0), (0, 0)])
        out.append((a, b))
    return out


def replay(rings, runs, seed):
    rng = random.Random(seed)
    for _ in range(runs):
        Block(pieces(rng), rings, rng).run()


def kernel_rings():
    text = open(os.path.join(ROOT, "lazyweights_b200", "csrc", "lw_attend_prompt.cu")).read()
    found = [re.search(r"%s = DP == 128 \? (\d+) : (\d+);" % name, text) for name in ("kKeyStages", "kValueStages")]
    return [tuple(int(f.group(i)) for f in found) for i in (1, 2)]


@pytest.mark.parametrize("dims", [0, 1])
def test_the_kernels_rings(dims):
    replay(kernel_rings()[dims], 1500, dims)


def test_one_ring_for_both_is_seen_to_fail():
    with pytest.raises(Overwritten):
        replay((5,), 1500, 3)


def test_a_block_that_gives_up_waits_for_every_copy():
    """Each barrier that copies are counted on is waited for before the block gives its shared memory back."""
    text = open(os.path.join(ROOT, "lazyweights_b200", "csrc", "lw_attend_prompt.cu")).read()
    kernel = text[text.index("    k_attend_prompt("):text.index(" k_attend_join(")]
    on = set(re.findall(r"mbar_expect\((\w+)", kernel))
    on |= set(re.findall(r"uint64_t\* const bar = cut \? &(\w+) : (\w+)", kernel)[0])
    assert on - {"bar"} == {"full", "q_full", "tail_full"}
    gives_up = kernel[kernel.index("// Every copy has been waited for"):]
    assert all(re.search(r"mbar_wait\(smem_addr\(&?%s\b" % name, gives_up) for name in on - {"bar"})
