"""The account of a cache's pages against a cache of plain lists: whatever is forked, written, cut and moved, every sequence reads its own tokens."""

import random

import pytest
import torch

import __graft_entry__ as entry

entry.ensure_built()

from tt_xla_amd import CachePages, copy_cache_blocks  # noqa: E402


class Model:
    """Pages with contents, and what every sequence should read."""

    def __init__(self, nb, bs, reserved=1):
        self.pages = CachePages(nb, bs, reserved)
        self.held = [[None] * bs for _ in range(nb)]
        self.want = {}

    def copy(self, pairs):
        for s, t in pairs:
            assert s != t and t >= self.pages.reserved
            self.held[t] = list(self.held[s])

    def write(self, s, first, tokens):
        bs = self.pages.block_size
        for i, x in enumerate(tokens, first):
            page = self.pages.pages(s)[i // bs]
            assert sum(page in self.pages.pages(o) for o in self.want) == 1  # nobody else's
            self.held[page][i % bs] = x
        self.want[s][first:] = tokens

    def check(self):
        bs, p = self.pages.block_size, self.pages
        used = set()
        for s, want in self.want.items():
            pages = p.pages(s)
            assert p.length(s) == len(want) and len(pages) == -(-len(want) // bs) and len(set(pages)) == len(pages)
            assert [self.held[pages[i // bs]][i % bs] for i in range(len(want))] == want
            used |= set(pages)
        assert not used & set(range(p.reserved)) and p.free_pages == p.num_blocks - p.reserved - len(used)


@pytest.mark.parametrize("seed", range(20))
def test_whatever_happens_everybody_reads_their_own(seed):
    r = random.Random(seed)
    m = Model(r.choice([6, 12, 40]), r.choice([1, 2, 5]), r.choice([0, 1, 3]))
    names, full = iter(range(10**6)), 0
    for _ in range(300):
        some = list(m.want)
        what = r.choice(["add", "extend", "extend", "fork", "rewrite", "cut", "free", "compact"])
        before = {s: (m.pages.pages(s), m.pages.length(s)) for s in some}, m.pages.free_pages
        try:
            if what == "add":
                s, n = next(names), r.randrange(9)
                m.pages.add(s, n)
                m.want[s] = []
                m.write(s, 0, [(s, i, r.random()) for i in range(n)])
            elif not some:
                continue
            else:
                s = r.choice(some)
                at = len(m.want[s])
                if what == "extend":
                    n = r.randrange(7)
                    m.copy(m.pages.extend(s, n))
                    m.write(s, at, [(s, i, r.random()) for i in range(n)])
                elif what == "fork":
                    c = next(names)
                    m.pages.fork(s, c)
                    m.want[c] = list(m.want[s])
                elif what == "rewrite":
                    first = r.randrange(at + 2)
                    m.copy(m.pages.own(s, first))
                    m.write(s, min(first, at), [(s, i, r.random()) for i in range(max(0, at - first))] if first < at else [])
                elif what == "cut":
                    n = r.randrange(at + 1)
                    m.pages.truncate(s, n)
                    del m.want[s][n:]
                elif what == "free":
                    m.pages.free(s)
                    del m.want[s]
                else:
                    pairs = m.pages.compact()
                    assert not {t for _, t in pairs} & {s for s, _ in pairs}  # no order among them
                    m.copy(pairs)
                    top = max((max(m.pages.pages(x), default=-1) for x in m.want), default=-1)
                    assert top < m.pages.num_blocks - m.pages.free_pages
        except RuntimeError:  # no pages left: nothing has changed
            full += 1
            assert ({s: (m.pages.pages(s), m.pages.length(s)) for s in some}, m.pages.free_pages) == before
        m.check()
    assert full or m.pages.num_blocks == 40


def test_tables_and_refusals():
    p = CachePages(10, 4)
    p.add("a", 6)
    p.add("none", 0)
    assert p.table(["a", "none"], 3).tolist() == [[1, 2, 0], [0, 0, 0]] and p.table(["a"], 3, fill=-1).tolist() == [[1, 2, -1]]
    p.fork("a", "b")
    assert p.extend("b", 3) == [(2, 3)] and p.pages("b") == [1, 3, 4] and p.extend("a", 1) == []
    assert p.own("a", 4) == [] and p.own("a") == [(1, 5)] and p.own("b") == []
    for error, call in ((ValueError, lambda: p.add("a", 1)), (ValueError, lambda: p.fork("a", "b")), (ValueError, lambda: p.truncate("a", 8)), (ValueError, lambda: p.extend("a", -1)),
                        (ValueError, lambda: p.own("a", -1)), (ValueError, lambda: p.add("c", -1)), (ValueError, lambda: p.table(["b"], 2)), (RuntimeError, lambda: p.extend("a", 100)),
                        (KeyError, lambda: p.free("nobody")), (ValueError, lambda: CachePages(0, 4)), (ValueError, lambda: CachePages(4, 4, 5))):
        with pytest.raises(error):
            call()
    with pytest.raises(RuntimeError):
        p.add("c", 100)
    with pytest.raises(KeyError):
        p.length("c")


def test_copies_name_blocks_that_exist():
    caches = {"a": [torch.zeros(4, 2, 8), torch.zeros(4, 2, 8)]}
    copy_cache_blocks(caches, [])
    copy_cache_blocks({}, [(0, 9)])
    for pair in ((0, 4), (-1, 2)):
        with pytest.raises(ValueError, match="outside"):
            copy_cache_blocks(caches, [pair])
