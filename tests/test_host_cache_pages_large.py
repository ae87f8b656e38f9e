"""The account of a large cache's pages: a page that goes back, or is taken, costs a few comparisons, however many pages are free."""

import random

import __graft_entry__ as entry

entry.ensure_built()

from tt_xla_amd import CachePages  # noqa: E402


class Counted(int):
    seen = 0

    def __lt__(self, other):
        Counted.seen += 1
        return int(self) < int(other)


def test_comparisons_of_a_step():
    nb, bs = 1 << 16, 4
    p = CachePages(nb, bs)
    p._free[:] = [Counted(x) for x in p._free]
    r, live, moved = random.Random(1), [], 0
    Counted.seen = 0
    for i in range(400):
        p.add(i, 30)
        live.append(i)
        moved += 8
        if i % 3 == 2:  # a fork, whose written page is replaced by a copy
            s = r.choice(live)
            p.fork(s, -i)
            moved += len(p.pages(s)) + len(p.extend(-i, 9)) + 3
            p.free(-i)
        if i % 2:
            s = live.pop(r.randrange(len(live)))
            moved += len(p.pages(s))
            p.free(s)
    # (a heap of 2^16: 16 levels, two comparisons each at most, for a page that is taken or given back)
    assert moved > 4000 and Counted.seen <= 2 * 16 * 2 * moved


def test_the_lowest_free_page_is_taken_next():
    p, r, free, live = CachePages(200, 1, 3), random.Random(2), set(range(3, 200)), {}
    for i in range(500):
        if live and (r.random() < 0.4 or len(free) < 8):
            s = r.choice(list(live))
            free |= set(live.pop(s))
            p.free(s)
        else:
            n = r.randrange(1, 8)
            p.add(i, n)
            want = sorted(free)[:n]
            assert p.pages(i) == want
            live[i] = want
            free -= set(want)
        if i % 97 == 96:
            moved = dict(p.compact())
            live = {s: [moved.get(x, x) for x in pages] for s, pages in live.items()}
            free = set(range(3, 200)) - {x for pages in live.values() for x in pages}
            assert all(p.pages(s) == pages for s, pages in live.items())
        assert p.free_pages == len(free)
