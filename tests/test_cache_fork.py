"""Sequences that share pages, and eight-bit requests: the cache's bookkeeping (no GPU)."""
import random

import pytest

from inferllm_b200.binding import CacheError, CacheFull
from inferllm_b200.cache import FixedState, PagedKV, SequenceCache


def cache(num_pages=20, slots=6, page=4, longest=64, requests=None):
    return SequenceCache(requests or {0: PagedKV(2, 8), 1: PagedKV(1, 16, int8=True)}, slots, num_pages, page, longest)


def grow(c, slots, q_lens):
    plan = c.plan_step(slots, q_lens)
    c.commit_step(plan)
    return plan


def test_a_fork_holds_the_same_pages_until_the_last_holder_ends():
    c = cache()
    a = c.alloc_slot()
    grow(c, [a], [10])
    free = c.pages_free()
    b = c.fork_slot(a, 8)
    assert c.pages_free() == free and c.seq_len[b] == 8
    for g in (0, 1):
        assert [c.pages_of(g, b)[i] for i in (0, 1)] == [c.pages_of(g, a)[i] for i in (0, 1)] and len(c.pages_of(g, b)) == 2
    plan = grow(c, [a, b], [1, 3])
    for g in (0, 1):
        tab = plan.tables[g]
        assert list(tab[0, :2]) == list(tab[1, :2]) and tab[0, 2] != tab[1, 2] and tab[1, 2] >= 0
    c.check()
    c.free_slot(a)
    c.check()
    assert c.pages_free() == [20 - 3, 20 - 3]           # what b holds: two shared pages and its own
    d = c.fork_slot(b, 8)
    c.free_slot(b)
    c.check()
    assert c.pages_free() == [18, 18]
    c.free_slot(d)
    c.check()
    assert c.pages_free() == [20, 20]


def test_common_prefixes_of_a_step():
    c = cache(num_pages=60, slots=8)
    a = c.alloc_slot()
    grow(c, [a], [13])
    b, d = c.fork_slot(a, 12), c.fork_slot(a, 8)
    e = c.alloc_slot()
    grow(c, [e], [5])
    f = c.fork_slot(e, 4)
    alone = c.alloc_slot()
    grow(c, [b, d, f, alone], [2, 2, 2, 2])
    assert sorted(c.common_prefixes([a, b, d, e, f, alone])) == sorted([(8, [0, 1, 2]), (4, [3, 4])])
    assert c.common_prefixes([b, a]) == [(12, [0, 1])]
    assert c.common_prefixes([d, alone, e]) == [] and c.common_prefixes([a]) == []
    g = c.fork_slot(b, 12)                                # a fork of a fork
    assert c.common_prefixes([g, a]) == [(12, [0, 1])]
    c.reset()
    c.check()
    assert c.pages_free() == [60, 60]


def test_an_abandoned_step_gives_back_its_own_pages_only():
    c = cache()
    a = c.alloc_slot()
    grow(c, [a], [8])
    b = c.fork_slot(a, 8)
    before = c.pages_free()
    plan = c.plan_step([a, b], [5, 5])
    c.abandon_step(plan)
    c.check()
    assert c.pages_free() == before and len(c.pages_of(0, a)) == 2 and len(c.pages_of(0, b)) == 2
    with pytest.raises(CacheFull):
        c.plan_step([a, b], [40, 40])
    c.check()


def test_refusals():
    c = cache(slots=2)
    a = c.alloc_slot()
    grow(c, [a], [10])
    for length in (0, -4, 3, 6, 12, 64):
        with pytest.raises(CacheError):
            c.fork_slot(a, length)
    for slot in (1, 5, -1):
        with pytest.raises(CacheError):
            c.fork_slot(slot, 4)
    for slots in ([a, 1], [a, 2], [-1, a], [2 ** 31 - 1, a]):
        with pytest.raises(CacheError, match="not live"):
            c.common_prefixes(slots)
    c.fork_slot(a, 4)
    with pytest.raises(CacheFull):
        c.fork_slot(a, 4)
    c.check()
    for requests in ({0: PagedKV(2, 8, window=16)}, {0: PagedKV(2, 8, chunk=16)}, {0: PagedKV(2, 8), 1: FixedState((4,))}, {0: FixedState((4,))}):
        w = cache(requests=requests)
        s = w.alloc_slot()
        grow(w, [s], [9])
        with pytest.raises(CacheError, match="cannot be shared"):
            w.fork_slot(s, 4)
        assert w.common_prefixes([s, w.alloc_slot()]) == []
        w.check()


def test_eight_bit_requests_form_groups_of_their_own():
    c = cache(requests={0: PagedKV(2, 8), 1: PagedKV(2, 8, int8=True), 2: PagedKV(2, 8), 3: PagedKV(2, 8, int8=True)})
    groups = c.stats()["paged"]
    assert [g["entries"] for g in groups] == [[0, 2], [1, 3]] and [g["request"].get("int8", False) for g in groups] == [False, True]
    with pytest.raises(CacheError, match="keys-only"):
        cache(requests={0: PagedKV(1, 8, keys_only=True, int8=True)})


@pytest.mark.parametrize("seed", range(6))
def test_random_lives(seed):
    rng = random.Random(seed)
    c, live = cache(num_pages=40, slots=10, page=4, longest=80), {}
    for _ in range(300):
        op = rng.random()
        try:
            if op < 0.2:
                s = c.alloc_slot()
                live[s] = 0
            elif op < 0.45 and live:
                s = rng.choice(list(live))
                if live[s] >= 4:
                    n = rng.randint(1, live[s] // 4) * 4
                    t = c.fork_slot(s, n)
                    live[t] = n
            elif op < 0.6 and live:
                s = rng.choice(list(live))
                c.free_slot(s)
                del live[s]
            elif live:
                some = rng.sample(list(live), rng.randint(1, len(live)))
                q = [rng.randint(1, 6) for _ in some]
                if any(live[s] + n > 80 for s, n in zip(some, q)):
                    continue
                plan = c.plan_step(some, q)
                if rng.random() < 0.2:
                    c.abandon_step(plan)
                else:
                    c.commit_step(plan)
                    for s, n in zip(some, q):
                        live[s] += n
        except CacheFull:
            pass
        c.check()
        for s, n in live.items():
            assert c.seq_len[s] == n
        # a page that two sequences hold is full in both, and at the same place
        where = {}
        for s in live:
            for lp, p in c.pages_of(0, s).items():
                where.setdefault(p, []).append((s, lp))
        for holders in where.values():
            assert len({lp for _, lp in holders}) == 1
            if len(holders) > 1:
                assert all((lp + 1) * 4 <= live[s] for s, lp in holders)
    c.reset()
    c.check()
    assert c.pages_free() == [40, 40]


@pytest.mark.parametrize("seed", range(8))
def test_common_prefixes_are_the_pages_that_all_hold(seed):
    """Forks of forks at any length, some of whose origins have ended: against a comparison page by page."""
    rng = random.Random(seed)
    c, live = cache(num_pages=400, slots=30, page=4, longest=120), []
    for _ in range(4):
        s = c.alloc_slot()
        grow(c, [s], [rng.randint(4, 100)])
        live.append(s)
    for _ in range(60):
        if len(live) > 25 or (len(live) > 6 and rng.random() < 0.25):
            c.free_slot(live.pop(rng.randrange(len(live))))
            continue
        s = rng.choice(live)
        t = c.fork_slot(s, rng.randint(1, int(c.seq_len[s]) // 4) * 4)
        if c.seq_len[t] < 110:
            grow(c, [t], [rng.randint(1, 9)])
        live.append(t)
        some = rng.sample(live, rng.randint(1, len(live)))
        pages = [[p for _, p in sorted(c.pages_of(0, s).items())] for s in some]
        groups = {}
        for i, p in enumerate(pages):
            groups.setdefault(p[0], []).append(i)
        want = []
        for m in groups.values():
            if len(m) > 1:
                n = 0
                while all(len(pages[i]) > n and pages[i][n] == pages[m[0]][n] for i in m):
                    n += 1
                want.append((4 * n, m))
        assert sorted(c.common_prefixes(some)) == sorted(want)
        c.check()
