"""A model of the barrier protocol of the many-row paged attention (byteprof_b200/csrc/paged_attn_tc.cu), run on the CPU
under random schedules: the loading warp, the issuing thread, the warp that looks through a block's values and clears some,
and the two softmax groups, over a ring of two K and two V tiles. Every ring tile is tagged with the block it holds, so that a
product over a refilled tile, or a clearing that hits another block's values, fails an assertion; so does a softmax group
that does not get what that warp found in the blocks of its segment (`lost`).

A segment is (blocks, what tile 0 sees of them, what tile 1 sees). The rule that the kernel relies on: every block in the
ring is used by at least one tile. An item that sees nothing has a block to itself (its rows are written as zeros) that no
tile uses: in the ring, nothing would hold the clearing warp and the refill of its slot together, and the last test
shows the model catching that."""

import random

import pytest
from test_i4tc_ring_protocol import Deadlock, MBar

SLOTS = 4


def run(segments, seed, unused_in_ring=False, slow_clear=8):
    rng = random.Random(seed)
    full = [MBar(1) for _ in range(SLOTS)]
    empty, s_full, o_done = ([MBar(1) for _ in range(2)] for _ in range(3))
    p_full = [MBar(5) for _ in range(2)]
    ring, lost = [None] * SLOTS, [[(-1, 0)] * 2 for _ in range(2)]
    found = [[rng.random() < 0.3 for _ in range(seg[0])] for seg in segments]  # blocks with a value to take out
    events, now, last_commit = [], [0], [0]
    outputs = [[], []]  # per tile: (segment, block) of the products with V, in order

    def later(fn):
        events.append((now[0] + rng.randint(1, 40), fn))

    def commit(fn):  # tcgen05.commit arrivals complete in issue order
        t = max(now[0] + rng.randint(1, 40), last_commit[0] + 1)
        last_commit[0] = t
        events.append((t, fn))

    def used(seg):
        n, u0, u1 = seg
        return n if unused_in_ring else min(n, max(u0, u1))

    def wait(bar, parity):
        while not bar.done(parity):
            yield

    def loader():
        t = issued = 0
        for seg in segments:
            for _ in range(used(seg)):
                for kv in range(2):
                    slot = issued % SLOTS
                    if t >= 2:
                        pair = t - 2 + kv
                        yield from wait(empty[pair & 1], (pair >> 1) & 1)
                    full[slot].expect_tx(1)

                    def land(slot=slot, tag=("KV"[kv], t)):
                        ring[slot] = tag
                        full[slot].complete_tx(1)
                    later(land)
                    issued += 1
                    yield
                t += 1

    def issuer():
        blk, pn = 0, [0, 0]

        def scores(i, at):
            tag, slot = ("K", at), 2 * (at & 1)
            assert ring[slot] == tag, "scores of a stale K tile"

            def done():
                assert ring[slot] == tag, "K tile refilled under the product"
                s_full[i].arrive()
            commit(done)

        def output(i, at, s, b):
            tag, slot = ("V", at), 2 * (at & 1) + 1
            assert ring[slot] == tag, "product with a stale V tile"
            outputs[i].append((s, b))

            def done():
                assert ring[slot] == tag, "V tile refilled under the product"
            commit(done)

        for s, seg in enumerate(segments):
            n, un = used(seg), seg[1:]
            if n == 0:
                continue
            yield from wait(full[(2 * blk) & 3], (blk >> 1) & 1)
            for i in range(2):
                if un[i] > 0:
                    scores(i, blk)
            commit(empty[blk & 1].arrive)
            for b in range(n):
                if b >= un[0] and b >= un[1]:
                    yield from wait(full[(2 * blk + 1) & 3], (blk >> 1) & 1)
                for i in range(2):
                    if b < un[i]:
                        yield from wait(p_full[i], pn[i] & 1)
                        pn[i] += 1
                        output(i, blk, s, b)
                        if b + 1 < un[i]:
                            scores(i, blk + 1)
                        else:
                            commit(o_done[i].arrive)
                if b + 1 < n:
                    commit(empty[(blk + 1) & 1].arrive)
                blk += 1

    def clearer():
        blk, pn, segs = 0, [0, 0], [0, 0]
        for s, seg in enumerate(segments):
            n, un = used(seg), seg[1:]
            for b in range(n):
                slot, tag = (2 * blk + 1) & 3, ("V", blk)
                yield from wait(full[slot], (blk >> 1) & 1)
                if b + 1 == seg[0] or found[s][b]:  # the sequence's end lies in the last block
                    for _ in range(rng.randint(1, slow_clear)):
                        assert ring[slot] == tag, "another block's values are cleared"
                        yield
                    assert ring[slot] == tag, "another block's values are cleared"
                if b + 1 < n:
                    yield from wait(full[(2 * blk + 2) & 3], ((blk + 1) >> 1) & 1)
                for i in range(2):
                    if b < un[i]:
                        if pn[i] > 0:
                            yield from wait(p_full[i], (pn[i] + 1) & 1)
                        pn[i] += 1
                        if found[s][b]:
                            e = lost[i][segs[i] & 1]
                            lost[i][segs[i] & 1] = (segs[i], min(e[1], b) if e[0] == segs[i] else b)
                        p_full[i].arrive()
                blk += 1
            for i in range(2):
                segs[i] += un[i] > 0

    def softmax(i):
        n = segs = 0
        for s, seg in enumerate(segments):
            for _ in range(seg[1 + i]):
                yield from wait(s_full[i], n & 1)
                for _ in range(rng.randint(0, 6)):
                    yield
                p_full[i].arrive(4)
                n += 1
            if seg[1 + i] > 0:
                yield from wait(o_done[i], segs & 1)
                yield from wait(p_full[i], (n - 1) & 1)
                for _ in range(rng.randint(0, 10)):
                    yield
                e = lost[i][segs & 1]
                mine = [b for b in range(seg[1 + i]) if found[s][b]]
                assert (e[1] if e[0] == segs else None) == (mine[0] if mine else None), "another segment's finding is read"
                segs += 1

    alive = [loader(), issuer(), clearer(), softmax(0), softmax(1)]
    slow = rng.choice(alive)
    for _ in range(400_000):
        if not alive and not events:
            want = [[(s, b) for s, seg in enumerate(segments) for b in range(seg[1 + i])] for i in range(2)]
            assert outputs == want
            return
        if events and (not alive or rng.random() < 0.3):
            events.sort(key=lambda e: e[0])
            t, fn = events.pop(0)
            now[0] = max(now[0], t)
            fn()
            continue
        role = rng.choice(alive)
        if role is slow and rng.random() < 0.8:
            continue
        try:
            next(role)
        except StopIteration:
            alive.remove(role)
        now[0] += 1
    raise Deadlock("no progress")


EMPTY = (1, 0, 0)
CASES = [
    [(1, 1, 1)] * 6, [(3, 2, 3), (1, 1, 0), (5, 4, 5), (1, 0, 1)], [(12, 12, 12), (2, 0, 2)], [EMPTY] * 7,
    [EMPTY] * 4 + [(3, 3, 3)], [(2, 2, 2)] + [EMPTY] * 5 + [(1, 1, 1), (4, 3, 4)], [(1, 1, 0), EMPTY, (1, 0, 1), EMPTY, (7, 6, 7)] * 2,
    [EMPTY, (1, 1, 1)] * 5,
]


@pytest.mark.parametrize("segments", CASES)
def test_no_tile_is_refilled_or_cleared_under_its_readers(segments):
    for seed in range(60):
        run(segments, seed)


def test_unused_blocks_in_the_ring_are_caught():
    failures = 0
    for segments in CASES[4:]:
        for seed in range(60):
            try:
                run(segments, seed, unused_in_ring=True, slow_clear=40)
            except (AssertionError, Deadlock):
                failures += 1
    assert failures > 0
