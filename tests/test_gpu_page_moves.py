"""Copies of blocks and compaction of sequences inside paged caches (``tt::copy_cache_blocks_``, ``tt::keep_cache_tokens_``): bytes move, so
every result is exact."""

import pytest
import torch

import __graft_entry__ as entry
import media_reference as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _noise(g, *shape, dtype=torch.bfloat16):
    size = torch.empty((), dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=g, dtype=torch.uint8).view(dtype)


def _same(got, want):
    return torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8))


def _ids(*x):
    return torch.tensor(x, dtype=torch.int32)


def _copied(caches, source, target):
    on = [c.cuda() for c in caches]
    torch.ops.tt.copy_cache_blocks_(on, source.cuda(), target.cuda())
    want = [c.clone() for c in caches]
    M.copy_blocks([w.view(torch.uint8) for w in want], source, target)
    assert all(_same(a, b) for a, b in zip(on, want)), [int((a.cpu().view(torch.uint8) != b.view(torch.uint8)).sum()) for a, b in zip(on, want)]


@pytest.mark.parametrize("shape, dtype", [((24, 8, 64, 128), torch.bfloat16), ((24, 2, 32, 64), torch.uint8), ((24, 1, 16, 576), torch.bfloat16), ((24, 3), torch.float32),
                                          ((24, 5, 7), torch.uint8), ((24, 2, 2, 64), torch.bfloat16), ((24, 1), torch.float8_e4m3fn), ((24, 40, 128, 128), torch.uint8)])
@pytest.mark.parametrize("pairs", [1, 3, 4, 11])
def test_disjoint_pairs(shape, dtype, pairs):
    g = torch.Generator().manual_seed(pairs)
    order = torch.randperm(24, generator=g)
    _copied([_noise(g, *shape, dtype=dtype) for _ in range(3)], order[:pairs], order[12 : 12 + pairs])


@pytest.mark.parametrize("many", [False, True])
def test_pairs_that_depend_on_each_other(many):
    """Chains, swaps by way of a third block, one target twice, blocks onto themselves, ids outside the cache: as if the pairs went in order."""
    g = torch.Generator().manual_seed(7)
    nb = 90
    lists = [((3, 5, 5), (5, 6, 3)), ((1, 2, 0), (0, 1, 2)), ((4, 5), (7, 7)), ((2, 2, 2), (2, 3, 2)), ((-1, 4, 100, 5), (3, -7, 2, 90)), ((5, 6), (5, 8)), ((0, 9, 1), (9, 1, 0))]
    for source, target in lists:
        s, t = _ids(*source), _ids(*target)
        if many:  # behind and in front of pairs that depend on nothing, more than a wavefront has lanes
            free = torch.randperm(70, generator=g).int() + 20
            s, t = torch.cat([free[:34], s, _ids(-3) .expand(31)]), torch.cat([free[34:68], t, _ids(3).expand(31)])
        _copied([_noise(g, nb, 2, 32, 64), _noise(g, nb, 2, dtype=torch.float32)], s, t)
    # and any pairs at all
    n = 200 if many else 30
    _copied([_noise(g, nb, 3, 16, 64)], torch.randint(-2, nb + 2, (n,), generator=g), torch.randint(-2, nb + 2, (n,), generator=g))


def test_long_lists_and_large_caches():
    """More pairs than one launch takes, in order across launches; more blocks than a workgroup can mark."""
    g = torch.Generator().manual_seed(8)
    _copied([_noise(g, 300, 1, 16)], torch.randint(0, 300, (9001,), generator=g), torch.randint(0, 300, (9001,), generator=g))
    nb = (1 << 18) + 100
    order = torch.randperm(nb, generator=g)
    _copied([_noise(g, nb, 16, dtype=torch.uint8)], order[:150], order[150:300])
    chain = torch.arange(nb - 130, nb - 1)
    _copied([_noise(g, nb, 16, dtype=torch.uint8)], chain, chain + 1)


def test_many_caches_of_several_sizes():
    g = torch.Generator().manual_seed(9)
    caches = [_noise(g, 10, 2, 32, 64) for _ in range(200)] + [_noise(g, 10, 2, dtype=torch.float32) for _ in range(5)] + [_noise(g, 10, 2, 2, 64)]
    _copied(caches, torch.tensor([1, 2, 3]), torch.tensor([9, 8, 7]))


def test_blocks_beyond_four_gibibytes():
    cache = torch.zeros(20000, 8, 128, 128, dtype=torch.bfloat16, device="cuda")
    cache[19999], cache[1] = 3.0, 5.0
    torch.ops.tt.copy_cache_blocks_([cache], _ids(19999, 1).cuda(), _ids(2, 19998).cuda())
    assert bool((cache[2] == 3).all()) and bool((cache[19998] == 5).all()) and bool((cache[3:19998] == 0).all())
    table = torch.tensor([[19997, 19996]], dtype=torch.int32, device="cuda")
    cache[19996, :, 127] = 9.0
    torch.ops.tt.keep_cache_tokens_([cache], table, torch.tensor([[255]], device="cuda"), torch.tensor([1], device="cuda"))
    assert bool((cache[19997, :, 0] == 9).all()) and bool((cache[19997, :, 1:] == 0).all())


def test_copy_refusals():
    c = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    op, i = torch.ops.tt.copy_cache_blocks_, _ids(1).cuda()
    for args in [([c, c], i, i), ([c, c.view(8, 16, 64)[:4]], i, i), ([c, torch.zeros(5, 3, device="cuda")], i, i), ([c.transpose(0, 1)], i, i), ([c], i, _ids(1, 2).cuda()),
                 ([c], i.float(), i), ([c], i[None], i[None])]:
        with pytest.raises(ValueError):
            op(*args)
    for args in [([c], i.cpu(), i), ([c, torch.zeros(4, 2)], i, i), ([c.clone().requires_grad_()], i, i)]:
        with pytest.raises((NotImplementedError, ValueError)):
            op(*args)
    with pytest.raises((ValueError, NotImplementedError)):
        op([], i, i)
    op([c], i[:0], i[:0])
    op([torch.zeros(4, 0, device="cuda")], i, i)


# --------------------------------------------------------------------------- #
# compaction
# --------------------------------------------------------------------------- #
def _kept(caches, table, kept, lens, first=None):
    on = [c.cuda() for c in caches]
    args = [t.cuda() for t in (table, kept, lens)] + ([] if first is None else [first.cuda()])
    torch.ops.tt.keep_cache_tokens_(on, *args)
    for a, c in zip(on, caches):
        assert _same(a, M.keep_tokens(c, table, kept, lens, first))


@pytest.mark.parametrize("heads, bs, d", [(2, 32, 64), (8, 64, 128), (1, 16, 576), (3, 5, 8), (2, 32, 256), (1, 64, 40)])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.95, 1.0])
@pytest.mark.parametrize("tokens", [1, 20, 300, 1100])
def test_chosen_tokens(heads, bs, d, share, tokens):
    g = torch.Generator().manual_seed(tokens + d)
    users, width = 3, -(-tokens // bs) + 1
    table = torch.randperm(users * width + 2, generator=g)[: users * width].view(users, width).int()
    caches = [_noise(g, users * width + 2, heads, bs, d) for _ in range(3)]
    first = torch.tensor([0, tokens // 3, max(0, tokens - 9)])
    lens = torch.tensor([max(1, int((tokens - int(f)) * share)) for f in first])
    lens[1] = lens[1] if tokens != 20 else 0
    kept = torch.full((users, int(lens.max())), 1 << 30, dtype=torch.int32)
    for u in range(users):
        some = torch.randperm(tokens - int(first[u]), generator=g)[: int(lens[u])].sort().values + first[u]
        kept[u, : len(some)] = some.int()
    _kept(caches, table, kept, lens, first)
    _kept([c.view(torch.float16) for c in caches], table.long(), kept.long(), lens.int(), first.int())


@pytest.mark.parametrize("n", [5, 40, 700])
def test_entries_that_are_skipped(n):
    """Entries in any order, in front of their place, negative, outside the table or in pages outside the cache; lengths below zero and beyond the entries."""
    g = torch.Generator().manual_seed(n)
    users, bs, width = 4, 16, 50
    table = torch.randperm(users * width, generator=g).view(users, width).int()
    table[0, 3], table[1, 0], table[1, 40] = -1, users * width, 1 << 30
    caches = [_noise(g, users * width, 2, bs, 64)]
    kept = torch.randint(-5, width * bs + 60, (users, n), generator=g)
    kept[2] = torch.randint(-(1 << 40), 1 << 40, (n,), generator=g)
    lens, first = torch.tensor([n, n + 9, n, -3]), torch.tensor([0, 17, 5, 0])
    _kept(caches, table, kept, lens, first)
    _kept(caches, table, kept, lens)
    _kept(caches, table, kept, lens, torch.tensor([-4, 1 << 40, width * bs - 2, -(1 << 40)]))


def test_nothing_to_keep():
    c = torch.ones(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    i = dict(dtype=torch.int32, device="cuda")
    torch.ops.tt.keep_cache_tokens_([c], torch.zeros(0, 2, **i), torch.zeros(0, 3, **i), torch.zeros(0, **i))
    torch.ops.tt.keep_cache_tokens_([c], torch.zeros(1, 2, **i), torch.zeros(1, 0, **i), torch.ones(1, **i))
    torch.ops.tt.keep_cache_tokens_([c], torch.zeros(1, 2, **i), torch.zeros(1, 3, **i), torch.zeros(1, **i))
    assert bool((c == 1).all())


def test_keep_refusals():
    z = dict(device="cuda")
    c = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, **z)
    t, k, n = torch.zeros(2, 3, dtype=torch.int32, **z), torch.zeros(2, 5, dtype=torch.int32, **z), torch.zeros(2, dtype=torch.int32, **z)
    op = torch.ops.tt.keep_cache_tokens_
    for args in [([c, c], t, k, n), ([c, torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, **z)], t, k, n), ([c[0]], t, k, n), ([c], t[0], k, n), ([c], t, k[:1], n),
                 ([c], t, k, n[:1]), ([c], t, k, n, n[:1]), ([c], t, k.float(), n), ([c], t.float(), k, n), ([c], t, k, n.float())]:
        with pytest.raises(ValueError):
            op(*args)
    for dtype in (torch.uint8, torch.float8_e4m3fn, torch.float32):
        with pytest.raises(NotImplementedError, match="rows"):
            op([torch.zeros(4, 2, 16, 64, dtype=torch.uint8, **z).view(dtype) if dtype.itemsize == 1 else c.float()], t, k, n)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        op([torch.zeros(4, 2, 16, 12, dtype=torch.bfloat16, **z)], t, k, n)
    with pytest.raises(NotImplementedError):
        op([c], t, k.cpu(), n)


def test_captured_moves():
    """Copies and a compaction in one graph, replayed with other pairs and tokens; every replay against the eager calls."""
    g = torch.Generator().manual_seed(12)
    state = [_noise(g, 40, 2, 16, 64).cuda() for _ in range(4)]
    source, target = _ids(*range(10)).cuda(), _ids(*range(10, 20)).cuda()
    table = torch.arange(20, 40).view(2, 10).int().cuda()
    kept, lens, first = torch.zeros(2, 60, dtype=torch.int32).cuda(), _ids(0, 0).cuda(), _ids(0, 0).cuda()

    def run(caches):
        torch.ops.tt.copy_cache_blocks_(caches, source, target)
        torch.ops.tt.keep_cache_tokens_(caches, table, kept, lens, first)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run([c.clone() for c in state])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(state)
    for n in range(4):
        source.copy_(torch.randint(0, 40, (10,), generator=g))
        target.copy_(torch.randint(0, 40, (10,), generator=g))
        kept.copy_(torch.stack([torch.randperm(160, generator=g)[:60].sort().values for _ in range(2)]))
        lens.copy_(_ids(60 - n, 7 * n))
        copy = [c.clone() for c in state]
        graph.replay()
        run(copy)
        if n % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state, copy))
