"""The hand-overs between the warps of `chunk_attn_tc_kernel`, as a model on the CPU: every role with the barriers it
waits for, the copies and the MMAs complete after random delays, and the roles run at random speeds.  A phase of an
mbarrier is told by one bit, as on the device; a named barrier counts arrivals and has no limit.

Two things are held: however the roles are scheduled they all come to an end (no phase of a barrier is overtaken by the
one after the next), and they do so, too, when a wait gives up anywhere (no warp is left behind at a barrier without a
limit).  Mistakes planted in the model show that it notices either.
"""
import random

import pytest

RING, SLOTS = 5, 4


class Stuck(AssertionError):
    pass


class Mbar:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return (self.phase & 1) != parity


class Named:
    """bar.sync / bar.red of `n` warps; `why` tells for what they came: two reasons at once means that they drifted."""

    def __init__(self, n):
        self.n, self.arrived, self.round, self.any = n, [], 0, False

    def meet(self, why, x=False):
        self.arrived.append((why, x))
        mine = self.round
        if len(self.arrived) == self.n:
            if len({w for w, _ in self.arrived}) > 1:
                raise Stuck(("warps meet for different reasons", self.arrived))
            self.any, self.arrived, self.round = any(x for _, x in self.arrived), [], self.round + 1
        while self.round == mine:
            yield
        return self.any


class Reader:
    """A role's place in the list of pieces."""

    def __init__(self, k):
        self.k, self.slot, self.parity = k, 0, 0

    def peek(self):
        ok = yield from self.k.wait(self.k.piece_full[self.slot], self.parity)
        return self.k.slots[self.slot] if ok else None

    def pop(self):
        self.k.piece_empty[self.slot].arrive()
        self.slot += 1
        if self.slot == SLOTS:
            self.slot, self.parity = 0, self.parity ^ 1


class Kernel:
    """One CTA's run.  pieces: for either block, which of the piece's tiles it sees.  Two softmax warps (one pair) a block."""

    def __init__(self, pieces, seed, fp16=False, give_up=0.0, hand_over_all=False, agree=True):
        self.rng, self.pieces, self.fp16, self.give_up = random.Random(seed), pieces, fp16, give_up
        self.hand_over_all, self.agree, self.aborted = hand_over_all, agree, False
        self.full, self.empty = [Mbar(1) for _ in range(RING)], [Mbar(2) for _ in range(RING)]
        self.s_ready, self.o_done, self.my_turn, self.drained = ([Mbar(1), Mbar(1)] for _ in range(4))
        self.p_ready, self.q_ready, self.pair_move = ([Mbar(2), Mbar(2)] for _ in range(3))
        self.piece_full, self.piece_empty = [Mbar(1) for _ in range(SLOTS)], [Mbar(7) for _ in range(SLOTS)]
        self.slots, self.pair, self.end = [None] * SLOTS, [Named(2), Named(2)], Named(8)
        self.mmas, self.copies, self.s_move = ([], []), [], [None, None]
        self.begin_tiles = [self.rng.choice([1, 1, 1, 2, 3]) for _ in range(5)]  # tiles until all rows have a reference point

    def wait(self, bar, parity):
        if not self.aborted and self.rng.random() < self.give_up:
            self.aborted = True
            return False
        while not bar.passed(parity):
            yield
            if self.aborted and self.rng.random() < 0.2:
                return False
        return True

    def idle(self):
        for _ in range(self.rng.randrange(4)):
            yield

    def softmax(self, blk):
        read, pair, live, seen, finished, moves = Reader(self), self.pair[blk], True, 0, 0, 0

        def hand_q(piece):
            if piece is not None and (self.hand_over_all or any(piece[1][blk])):
                self.q_ready[blk].arrive()

        hand_q((yield from read.peek()))
        while live:
            now = yield from read.peek()
            if (yield from pair.meet("top", now is None)):
                break
            read.pop()
            at, sees = now
            done = 0
            for i, see in enumerate(sees[blk]):
                if not see:
                    continue
                live = yield from self.wait(self.s_ready[blk], seen & 1)
                begins = done < self.begin_tiles[at % 5]
                if self.agree and begins:
                    live = not (yield from pair.meet(("live", at, i), not live))
                if self.agree and not live and (begins or not self.fp16):
                    break
                if begins:
                    yield from pair.meet(("maximum", at, i))
                if not self.fp16 and self.s_move[blk] == seen:
                    if self.agree:
                        for _ in range(2):
                            self.pair_move[blk].arrive()
                            live = yield from self.wait(self.pair_move[blk], moves & 1)
                            moves += 1
                            if not live:
                                break
                        if not live:
                            break
                    else:
                        yield from pair.meet(("move", at, i))
                yield from self.idle()
                if self.fp16:
                    if (yield from pair.meet(("too large", at, i), not live)):
                        live = not (yield from pair.meet(("live?", at, i), not live))
                elif self.rng.random() < 0.2:
                    self.s_move[blk] = seen + 1
                self.p_ready[blk].arrive()
                done, seen = done + 1, seen + 1
                if not live:
                    break
            live = not (yield from pair.meet(("tiles", at), not live))
            yield from pair.meet(("sums", at))
            following = (yield from read.peek()) if live else None
            if live and done:
                live = yield from self.wait(self.o_done[blk], finished & 1)
                finished += 1
            hand_q(following)
            live = not (yield from pair.meet(("output", at), not live))
            if live:
                yield from self.idle()
        yield from self.end.meet("end")

    def issuer(self, blk):
        read, turn, e, parity, seen, queries, issued = Reader(self), blk ^ 1, 0, 0, 0, 0, False
        ok = True
        while ok:
            now = yield from read.peek()
            if now is None:
                break
            read.pop()
            sees, n = now[1][blk], len(now[1][blk])
            last = max((i for i in range(n) if sees[i]), default=-1)
            if last >= 0 or self.hand_over_all:
                ok = (yield from self.wait(self.q_ready[blk], queries & 1)) and ok
                queries += 1
            ok = (yield from self.wait(self.full[e], parity)) and ok
            ok = (yield from self.wait(self.my_turn[blk], turn)) and ok
            self.mmas[blk].extend([self.s_ready[blk]] * sees[0] + [self.empty[e]])
            issued = True
            self.my_turn[blk ^ 1].arrive()
            turn ^= 1
            e, parity = (e + 1) % RING, parity ^ (e + 1 == RING)
            for i in range(n):
                if not ok:
                    break
                ve, vparity = e, parity
                e, parity = (e + 1) % RING, parity ^ (e + 1 == RING)
                more = i + 1 < n
                ok = (yield from self.wait(self.full[ve], vparity)) and ok
                if more:
                    ok = (yield from self.wait(self.full[e], parity)) and ok
                ok = (yield from self.wait(self.my_turn[blk], turn)) and ok
                if sees[i]:
                    ok = (yield from self.wait(self.p_ready[blk], seen & 1)) and ok
                self.mmas[blk].extend([self.o_done[blk]] * (i == last) + [self.empty[ve]])
                self.mmas[blk].extend([self.s_ready[blk]] * (more and sees[i + 1]))
                self.my_turn[blk ^ 1].arrive()
                turn ^= 1
                if more:
                    self.mmas[blk].append(self.empty[e])
                    e, parity = (e + 1) % RING, parity ^ (e + 1 == RING)
                seen += sees[i]
        if issued:
            self.mmas[blk].append(self.drained[blk])
            while not self.drained[blk].passed(0):
                yield
        yield from self.end.meet("end")

    def loader(self, is_v):
        read, e, parity, slot, slot_parity, live, left = Reader(self), is_v, 1, 0, 1, True, list(enumerate(self.pieces))
        while live:
            if is_v:
                now = yield from read.peek()
                if now is None:
                    break
                read.pop()
            else:
                now = left.pop(0) if left else None
                if not (yield from self.wait(self.piece_empty[slot], slot_parity)):
                    break
                self.slots[slot] = now
                self.piece_full[slot].arrive()
                slot, slot_parity = (slot + 1) % SLOTS, slot_parity ^ (slot + 1 == SLOTS)
                if now is None:
                    break
            for _ in now[1][0]:
                live = yield from self.wait(self.empty[e], parity)
                if not live:
                    break
                self.copies.append(self.full[e])
                e, parity = (e + 2) % RING, parity ^ (e + 2 >= RING)
        yield from self.end.meet("end")

    def state(self):
        bars = (self.full, self.empty, self.s_ready, self.o_done, self.my_turn, self.drained, self.p_ready, self.q_ready,
                self.pair_move, self.piece_full, self.piece_empty)
        return [(b.phase, b.pending) for group in bars for b in group] + [(n.round, len(n.arrived)) for n in self.pair + [self.end]]

    def run(self):
        roles = [(f(x), self.rng.choice([0.05, 0.3, 1.0])) for f, x in (
            (self.softmax, 0), (self.softmax, 0), (self.softmax, 1), (self.softmax, 1), (self.issuer, 0), (self.issuer, 1),
            (self.loader, 0), (self.loader, 1))]
        before, same = None, 0
        while roles:
            for done in (self.mmas[0], self.mmas[1]):  # in the order of issue
                if done and self.rng.random() < 0.3:
                    done.pop(0).arrive()
            if self.copies and self.rng.random() < 0.5:  # in any order
                self.copies.pop(self.rng.randrange(len(self.copies))).arrive()
            for role in list(roles):
                if self.rng.random() < role[1] and next(role[0], self) is self:
                    roles.remove(role)
            now = self.state() + [len(roles)]
            same = same + 1 if now == before else 0
            before = now
            if same > 2000:
                raise Stuck("nobody moves")


def _row_tile(n0, n1, skip=0):
    """A row tile: block 0 sees n0 tiles, block 1 all but the first `skip` of n1."""
    n = max(n0, n1, 1)
    return [[i < n0 for i in range(n)], [skip <= i < n1 for i in range(n)]]


RUNS = {
    "one tile, one block": [_row_tile(1, 0)] * 7,
    "two tiles, one block": [_row_tile(2, 0)] * 5,
    "two without the second block, then one with it": [_row_tile(1, 0), _row_tile(1, 0), _row_tile(1, 1), _row_tile(2, 0)] * 3,
    "nothing seen": [_row_tile(0, 0), _row_tile(1, 0), _row_tile(0, 0), _row_tile(0, 0), _row_tile(2, 2)] * 2,
    "windows": [_row_tile(4, 5, 1), _row_tile(6, 7, 2), _row_tile(3, 4, 1)],
    "long": [_row_tile(25, 26), _row_tile(9, 9)],
}


@pytest.mark.parametrize("name", RUNS)
def test_every_run_ends(name):
    for seed in range(25):
        Kernel(RUNS[name], seed, fp16=seed % 2 == 1).run()


@pytest.mark.parametrize("name", RUNS)
def test_every_run_ends_when_a_wait_gives_up(name):
    for seed in range(60):
        Kernel(RUNS[name], seed, fp16=seed % 2 == 1, give_up=(0.002, 0.01, 0.05)[seed % 3]).run()


def test_the_model_notices_an_overtaken_phase():
    """Q handed over for every piece: the softmax of a block that sees nothing is two phases ahead of its issuer."""
    with pytest.raises(Stuck):
        for seed in range(25):
            Kernel(RUNS["one tile, one block"], seed, hand_over_all=True).run()


def test_the_model_notices_a_warp_left_behind():
    """The two warps of a row do not tell each other that one gave up."""
    with pytest.raises(Stuck):
        for seed in range(300):
            Kernel(RUNS["long"], seed, give_up=0.01, agree=False).run()
