"""The barriers between the roles of the paged attention's tiles form, walked through on the
CPU: every order in which the roles of a CTA with two softmax groups can run.

An mbarrier wait names a phase by its parity alone: it passes while the barrier is in any
phase of the other parity.  It means "phase k is complete" only where phase k - 1 is known
to be complete and phase k + 1 cannot be.  The model counts phases, so it sees a wait that
passes for a phase that is still open; and it keeps track of the products, so it sees a warp
that touches O, P or the scores while a product still uses them.

What is modelled: two groups of two warps each (32 rows a warp, the groups take the units in
turn), the issuers of S (one per parity) and of P V, and the tensor pipe, which finishes the
products of an issuer in order but late.  Whether a warp's maxima grow at a unit (a rescale
of O) is free at every unit.  The number of barriers in the pv_done ring is read from the
source; the smaller ring shows that the model can tell the difference."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(__file__), "..", "thunderllamax_b200", "csrc", "paged_tiles.cu")


class Model:
    """items: units of each item; edges: units with a bad-value pass after their product."""

    def __init__(self, items, ring, edges=(), warps=2):
        self.n, self.ring, self.edges, self.warps = sum(items), ring, set(edges), warps
        self.begin, self.last, at = [], [], 0
        for k in items:
            self.begin.append(at)
            at += k
            self.last.append(at - 1)
        self.need, self.names = [], {}
        self.programs = [self.softmax(g, w) for g in (0, 1) for w in range(warps)]
        self.programs += [self.qk(0), self.qk(1), self.pv()]
        self.problems = set()

    # barriers: (name, index) -> number; arrivals that complete a phase
    def bar(self, name, index, count):
        key = (name, index)
        if key not in self.names:
            self.names[key] = len(self.need)
            self.need.append(count)
        return self.names[key]

    def s_full(self, i):
        return self.bar("s_full", i & 1, 1), i >> 1

    def s_free(self, i):
        return self.bar("s_free", i & 1, self.warps), i >> 1

    def p_full(self, i):
        return self.bar("p_full", i & 1, self.warps), i >> 1

    def pv_done(self, i):
        return self.bar("pv_done", i % self.ring, 1), i // self.ring

    def m_full(self, w, i):
        return self.bar("m_full", (w, i & 1), 1), i >> 1

    def turn(self, i):
        return self.bar("turn", i & 1, 1), i >> 1

    def q_full(self, item):
        return self.bar("q_full", 0, 2 * self.warps), item

    def o_free(self, item):
        return self.bar("o_free", 0, 2 * self.warps), item

    def l_full(self, w, item):
        return self.bar("l_full", w, 2), item

    # the roles' programs: (op, ...) in order
    def softmax(self, g, w):
        p = []
        for item in range(len(self.begin) + 1):
            more = item < len(self.begin)
            if item > 0:
                last = self.last[item - 1]
                if more:
                    if (last & 1) != g:
                        p.append(("wait", *self.s_full(last)))
                    p.append(("q", last))                   # Q of the last item is overwritten
                    p.append(("arrive", *self.q_full(item)))
                if (last & 1) != g:
                    p.append(("wait", *self.m_full(w, last)))
                p.append(("arrive", *self.l_full(w, item - 1)))
                p.append(("wait", *self.l_full(w, item - 1)))
                p.append(("wait", *self.pv_done(last)))
                p.append(("o", last + 1))                   # O is read: products 0 .. last and no more
                p.append(("arrive", *self.o_free(item - 1)))
            elif more:
                p.append(("arrive", *self.q_full(0)))
            if not more:
                break
            for i in range(self.begin[item], self.last[item] + 1):
                if (i & 1) != g:
                    continue
                p.append(("wait", *self.s_full(i)))
                p.append(("s", i))
                p.append(("arrive", *self.s_free(i)))
                if i > 0:
                    p.append(("wait", *self.m_full(w, i - 1)))
                if i > self.begin[item]:
                    p.append(("maybe", 4))                  # a rescale, or past it
                    p.append(("wait", *self.pv_done(i - 1)))
                    p.append(("o", i))                      # read ...
                    p.append(("o", i))                      # ... and written back
                if i not in self.edges:
                    p.append(("arrive", *self.m_full(w, i)))
                if i >= 2:
                    p.append(("wait", *self.pv_done(i - 2)))
                    p.append(("p", i - 2))                  # the P buffer of unit i - 2 is written
                p.append(("arrive", *self.p_full(i)))
                if i in self.edges:
                    p.append(("wait", *self.pv_done(i)))
                    p.append(("o", i + 1))
                    p.append(("o", i + 1))
                    p.append(("arrive", *self.m_full(w, i)))
        return p

    def qk(self, b):
        p, item = [], 0
        for i in range(self.n):
            starts = i in self.begin
            item += starts and i > 0
            if (i & 1) != b:
                continue
            if i >= 2:
                p.append(("wait", *self.s_free(i - 2)))
            if i > 0:
                p.append(("wait", *self.turn(i - 1)))
            if starts:
                p.append(("wait", *self.q_full(item)))
            p.append(("issue_s", i))
            p.append(("arrive", *self.turn(i)))
        return p

    def pv(self):
        p, item = [], 0
        for i in range(self.n):
            if i in self.begin and i > 0:
                p.append(("wait", *self.o_free(item)))
                item += 1
            p.append(("wait", *self.p_full(i)))
            p.append(("issue_pv", i))
        return p

    # a state: program counters, (phases, arrivals) of the barriers, S and PV issued and complete
    def run(self, limit=4_000_000):
        for i in range(self.n):                             # number the barriers that only the pipe arrives at
            self.s_full(i), self.pv_done(i)
        start = ((0,) * len(self.programs), ((0, 0),) * len(self.need), (0, 0, 0, 0))
        seen, todo = {start}, [start]
        while todo:
            state = todo.pop()
            after = list(self.steps(state))
            if not after and any(pc < len(p) for pc, p in zip(state[0], self.programs)):
                self.problems.add("deadlock")
            for s in after:
                if s not in seen:
                    seen.add(s)
                    todo.append(s)
            assert len(seen) < limit
        return self.problems

    def arrive(self, bars, b):
        c, a = bars[b]
        a += 1
        new = (c + 1, 0) if a == self.need[b] else (c, a)
        return bars[:b] + (new,) + bars[b + 1:]

    def steps(self, state):
        pcs, bars, (s_out, s_done, v_out, v_done) = state
        pipe = (s_out, s_done, v_out, v_done)
        if s_done < s_out:                                  # the pipe finishes an S, or a P V
            yield pcs, self.arrive(bars, self.s_full(s_done)[0]), (s_out, s_done + 1, v_out, v_done)
        if v_done < v_out:
            yield pcs, self.arrive(bars, self.pv_done(v_done)[0]), (s_out, s_done, v_out, v_done + 1)
        for r, (pc, prog) in enumerate(zip(pcs, self.programs)):
            if pc == len(prog):
                continue
            step = lambda k=1: pcs[:r] + (pc + k,) + pcs[r + 1:]
            op, *x = prog[pc]
            if op == "wait":
                b, phase = x
                done = bars[b][0]
                if (done & 1) != (phase & 1):               # all that the hardware compares
                    if done <= phase:
                        self.problems.add("stale phase")
                    yield step(), bars, pipe
            elif op == "arrive":
                if bars[x[0]][0] != x[1]:
                    self.problems.add("arrival in another phase")
                yield step(), self.arrive(bars, x[0]), pipe
            elif op == "maybe":
                yield step(), bars, pipe
                yield step(x[0]), bars, pipe
            elif op == "o":                                 # O holds products 0 .. x - 1, none is running
                if v_done != x[0] or v_out != x[0]:
                    self.problems.add("O in use")
                yield step(), bars, pipe
            elif op == "p":
                if v_done <= x[0]:
                    self.problems.add("P in use")
                yield step(), bars, pipe
            elif op == "s":                                 # S(i) is there and not overwritten
                if s_done <= x[0] or s_out > x[0] + 2:
                    self.problems.add("S in use")
                yield step(), bars, pipe
            elif op == "q":
                if s_done <= x[0] or s_out != x[0] + 1:
                    self.problems.add("Q in use")
                yield step(), bars, pipe
            elif op == "issue_s":
                if s_out != x[0]:
                    self.problems.add("S out of turn")
                yield step(), bars, (s_out + 1, s_done, v_out, v_done)
            elif op == "issue_pv":
                yield step(), bars, (s_out, s_done, v_out + 1, v_done)


def ring_of_source():
    src = open(SRC).read()
    m = re.search(r"constexpr int kPvRing = (\d+);", src)
    # every use of the barriers goes through the ring's helpers
    uses = set(re.findall(r"pv_done\[([^\]]*)\]", src))
    ring = int(m.group(1)) if m else 2
    assert not m or uses <= {"i", "unit % kPvRing"}, uses
    return ring


@pytest.mark.parametrize("items,edges", [((9,), ()), ((5, 2), (4,)), ((1, 4, 2), ()), ((2, 1, 3), (1, 2))])
def test_two_groups_hand_off(items, edges):
    assert Model(items, ring_of_source(), edges).run() == set()


def test_the_model_sees_a_stale_phase():
    # two barriers in turn: a rescale at unit i can pass its wait for product i - 1 while i - 3 is open
    assert {"stale phase", "O in use"} <= Model((4,), 2).run()
