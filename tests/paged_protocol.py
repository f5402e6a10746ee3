"""The roles of the paged attention kernels and their barriers, restated on the host: of one CTA
of attn_paged_tc_kernel (csrc/attention_paged_tc.cu) the producer, the widening warps, the softmax
and MMA warps of both sides; of one of attn_paged_kernel (csrc/attention_paged.cu) the producer
and the four consumer warps.  Roles are generators, copies and matrix products agents that end at
any later time, and any wait may give up.

A run checks what the kernel's order rests on: no wait tells two phases apart wrongly, every read
finds the tile that it is meant to, rows go out only when their products are complete, every role
ends, and nothing is in flight when the last one has."""
from __future__ import annotations

import random


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.tx, self.done = count, count, 0, 0

    def _settle(self):
        if self.pending == 0 and self.tx == 0:
            self.done += 1
            self.pending = self.count

    def arrive(self, tx=0):
        assert self.pending > 0, "more arrivals than the barrier counts"
        self.tx += tx
        self.pending -= 1
        self._settle()

    def complete(self):
        self.tx -= 1
        self._settle()

    def passed(self, k):
        """The parity wait for the k-th completion (k = -1: a fresh barrier passes)."""
        assert k <= self.done <= k + 1, f"a wait for phase {k} at {self.done}: two phases apart"
        return (self.done & 1) != (k & 1)


class Run:
    """What the two kernels' CTAs have in common."""

    def __init__(self, items, rng, give_up):
        self.items, self.rng, self.give_up = items, rng, give_up
        self.copies = []          # (barrier, where, what)
        self.mem = {}             # what is where
        self.stored = {}

    def copy(self, bar, where, what):
        self.mem[where] = None
        bar.arrive(tx=1)
        self.copies.append((bar, where, what))

    def agents(self):
        return [("copy", i) for i in range(len(self.copies))]

    def agent(self, kind, i):
        bar, where, what = self.copies.pop(i)
        self.mem[where] = what
        bar.complete()

    def run(self):
        """Whether a wait gave up.  Roles and agents go on in a random order."""
        roles = dict.fromkeys(self.roles())
        for r in list(roles):
            self._resume(roles, r, None)
        gave_up = False
        while roles:
            ready = [r for r, w in roles.items() if w is None or w[0].passed(w[1])]
            moves = [("role", r) for r in ready] + self.agents()
            late = [r for r, w in roles.items() if w is not None and len(w) == 2]
            if late and (not moves or self.rng.random() < self.give_up):
                assert self.give_up > 0, "every role waits for another"
                gave_up = True
                self._resume(roles, self.rng.choice(late), False)
            else:
                assert moves, "a wait for copies or products that were never issued"
                kind, *what = self.rng.choice(moves)
                if kind == "role":
                    self._resume(roles, what[0], True)
                else:
                    self.agent(kind, what[0])
        assert not self.agents(), "something is in flight behind the last role"
        return gave_up

    def _resume(self, roles, r, answer):
        try:
            roles[r] = r.send(answer)
        except StopIteration:
            del roles[r]


class Cta(Run):
    """items: [(tiles, side B has rows)] of one CTA, in order."""

    def __init__(self, items, rng, give_up=0.0, forget_k=False):
        super().__init__(items, rng, give_up)
        self.forget_k = forget_k
        b = Barrier
        self.q_full, self.q_empty, self.a_turn = b(1), b(2), b(1)
        self.raw_full, self.raw_empty = [b(1), b(1)], [b(1), b(1)]
        self.full = [[b(1), b(1)], [b(1), b(1)]]    # K, V; stages
        self.empty = [[b(2), b(2)], [b(2), b(2)]]
        self.s_full, self.o_done, self.o_free, self.drain = ([b(1), b(1)] for _ in range(4))
        self.p_full = [[b(1), b(1)], [b(1), b(1)]]  # sides, halves
        self.queue = [[], []]     # of each side's MMA warp, in order
        # stored: (item, side) -> tiles in O

    def roles(self):
        return self.producer(), self.widen(), self.softmax(0), self.softmax(1), self.mma(0), self.mma(1)

    # ---- agents

    def agents(self):
        return super().agents() + [("mma", s) for s in (0, 1) if self.queue[s]]

    def agent(self, kind, i):
        if kind == "copy":
            super().agent(kind, i)
            return
        op = self.queue[i].pop(0)
        if op[0] == "commit":
            op[1].arrive()
        elif op[0] == "s":
            _, item, n = op
            assert self.mem["q"] == item and self.mem["wide", 0, n & 1] == n
            self.mem["s", i] = n
        else:
            _, n, half, start = op
            assert self.mem["wide", 1, n & 1] == n and self.mem["p", i, half] == n
            self.mem["o", i] = ([] if start else self.mem["o", i]) + [(n, half)]

    # ---- roles (yield a wait: the answer is whether it passed)

    def producer(self):
        n = n_k = items = 0
        ok = True
        for tiles, _ in self.items:
            ok = yield self.q_empty, items - 1
            if not ok:
                break
            self.copy(self.q_full, "q", items)
            for _ in range(tiles):
                for kv in (0, 1):
                    ok = yield self.raw_empty[kv], n - 1
                    if not ok:
                        break
                    n_k += kv == 0
                    self.copy(self.raw_full[kv], ("raw", kv), n)
                if not ok:
                    break
                n += 1
            items += 1
            if not ok:
                break
        if self.forget_k:
            n_k = n
        for bar, k in ((self.q_full, items), (self.raw_full[0], n_k), (self.raw_full[1], n)):
            if k:
                yield bar, k - 1, "drain"

    def widen(self):
        n = 0
        for tiles, _ in self.items:
            for _ in range(tiles):
                for kv in (0, 1):
                    st = n & 1
                    ok = yield self.raw_full[kv], n
                    ok = ok and (yield self.empty[kv][st], (n >> 1) - 1)
                    if not ok:
                        return
                    assert self.mem["raw", kv] == n
                    self.mem["wide", kv, st] = None
                    yield None
                    assert self.mem["raw", kv] == n
                    self.mem["wide", kv, st] = n
                    self.full[kv][st].arrive()
                    self.raw_empty[kv].arrive()
                n += 1

    def softmax(self, side):
        n = own = both = 0
        for item, (tiles, two) in enumerate(self.items):
            if side == 1 and not two:
                n += tiles
                continue
            first = n
            for _ in range(tiles):
                if not (yield self.s_full[side], own):
                    return
                assert self.mem["s", side] == n
                if side == 1 or (two and both > 0):
                    if not (yield (self.a_turn, both) if side else (self.p_full[1][1], both - 1)):
                        return
                assert self.mem["s", side] == n
                for half in (0, 1):
                    yield None
                    self.mem["p", side, half] = n
                    self.p_full[side][half].arrive()
                if side == 0 and two:
                    self.a_turn.arrive()
                n, own, both = n + 1, own + 1, both + two
            if not (yield self.o_done[side], own - 1):
                return
            want = [(i, half) for i in range(first, n) for half in (0, 1)]
            assert self.mem["o", side] == want
            yield None
            assert self.mem["o", side] == want
            self.stored[item, side] = tiles
            self.o_free[side].arrive()

    def mma(self, side):
        n = mine = own = 0
        put = self.queue[side].append
        busy = False

        def pv(i, start):
            if not (yield self.full[1][i & 1], i >> 1):
                return False
            if start and not (yield self.o_free[side], own - 1):
                return False
            for half in (0, 1):
                if not (yield self.p_full[side][half], mine - 1):
                    return False
                put(("pv", i, half, start and half == 0))
                if half:
                    put(("commit", self.o_done[side]))
                    put(("commit", self.empty[1][i & 1]))
            return True

        ok = True
        for item, (tiles, two) in enumerate(self.items):
            ok = yield self.q_full, item
            if side == 1 and not two:
                for _ in range(tiles):
                    ok = ok and (yield self.full[0][n & 1], n >> 1)
                    ok = ok and (yield self.full[1][n & 1], n >> 1)
                    if not ok:
                        break
                    self.empty[0][n & 1].arrive()
                    self.empty[1][n & 1].arrive()
                    n += 1
                if ok:
                    self.q_empty.arrive()
            else:
                for t in range(tiles):
                    ok = ok and (yield self.full[0][n & 1], n >> 1)
                    if ok and t > 0:
                        ok = yield from pv(n - 1, t == 1)
                    if ok and mine > 0:
                        ok = yield self.o_done[side], mine - 1
                    if not ok:
                        break
                    put(("s", item, n))
                    put(("commit", self.s_full[side]))
                    put(("commit", self.empty[0][n & 1]))
                    busy = True
                    n, mine = n + 1, mine + 1
                if not ok:
                    break
                put(("commit", self.q_empty))
                ok = yield from pv(n - 1, tiles == 1)
                own += 1
            if not ok:
                break
        if busy:
            put(("commit", self.drain[side]))
            yield self.drain[side], 0, "drain"


class FewRows(Run):
    """items: tiles of each.  forget: a warp whose wait ran out keeps its own rows back only."""

    STAGES, WARPS = 3, 4

    def __init__(self, items, rng, give_up=0.0, forget=False):
        super().__init__([t for t in items], rng, give_up)
        self.forget = forget
        self.full = [Barrier(1) for _ in range(self.STAGES)]
        self.empty = [Barrier(self.WARPS) for _ in range(self.STAGES)]
        self.meet = Barrier(self.WARPS)
        self.fail = False
        self.seen = {}            # item -> (warp, tile) that its sums hold
        self.kept = set()         # items whose rows were left as they were, or marked

    def roles(self):
        return [self.producer()] + [self.consumer(w) for w in range(self.WARPS)]

    def producer(self):
        n = issued = 0
        ok, st = True, self.STAGES
        for tiles in self.items:
            for base in range(0, tiles, 8):
                count, ahead = min(8, tiles - base), 0
                while n == 0 and ahead < min(count, st) and ok:
                    ok = yield self.empty[ahead % st], ahead // st - 1
                    if ok:
                        self._fetch(ahead)
                        ahead += 1
                for i in range(count):
                    if ok and i >= ahead:
                        ok = yield self.empty[n % st], n // st - 1
                        if ok:
                            self._fetch(n)
                    if not ok:
                        break
                    self._arrive(n)
                    n += 1
                issued = max(n, ahead)
                if not ok:
                    break
            if not ok:
                break
        for n in range(n, issued):
            self._arrive(n)
        n = max(n, issued)
        for j in range(max(n - st, 0), n):
            yield self.full[j % st], j // st, "drain"

    def _fetch(self, n):
        """Announces the bytes of a copy without arriving."""
        bar = self.full[n % self.STAGES]
        bar.tx += 1
        self.mem[n % self.STAGES] = None
        self.copies.append((bar, n % self.STAGES, n))

    def _arrive(self, n):
        self.full[n % self.STAGES].arrive()

    def consumer(self, w):
        n = met = 0
        ok = True
        for item, tiles in enumerate(self.items):
            sums = []
            for t in range(tiles):
                st = n % self.STAGES
                ok = ok and (yield self.full[st], n // self.STAGES)
                if ok:
                    assert self.mem[st] == n
                    yield None
                    assert self.mem[st] == n
                    sums.append((w, t))
                    self.empty[st].arrive()
                n += 1
            self.seen.setdefault(item, []).extend(sums)
            if not ok:
                self.fail = True
            self.meet.arrive()
            yield self.meet, met, "meet"
            met += 1
            if ok if self.forget else not self.fail:
                self.stored[item] = tiles
                want = sorted((v, t) for v in range(self.WARPS) for t in range(tiles))
                assert sorted(self.seen[item]) == want, "rows without all of their keys"
            else:
                self.kept.add(item)
            self.meet.arrive()
            yield self.meet, met, "meet"
            met += 1


def random_items(rng):
    """Items of a share: a few tiles each, some without rows for side B."""
    two = rng.choice([0.0, 0.5, 0.9, 1.0])
    return [(rng.choice([1, 1, 2, 3, rng.randint(1, 7)]), rng.random() < two) for _ in range(rng.randint(1, 9))]
