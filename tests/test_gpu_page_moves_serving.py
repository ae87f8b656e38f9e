"""Copies of blocks and compaction of sequences as they are laid out for a serving batch: several caches per wavefront, whole rows per workgroup, more caches than a launch takes, several
trips through the pairs.  Bytes move, so every result is exact."""

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


def _kept(g, caches, table, counts, tokens, first, most):
    """Chosen ones of every user's tokens from `first` on move together; against the plain form, byte for byte."""
    users = table.shape[0]
    kept = torch.full((users, most), -1, dtype=torch.int32)
    for u, n in enumerate(counts):
        kept[u, :n] = (torch.randperm(tokens - first[u], generator=g)[:n].sort().values + first[u]).int()
    on = [c.cuda() for c in caches]
    lens, start = torch.tensor(counts, dtype=torch.int32), torch.tensor(first, dtype=torch.int32)
    torch.ops.tt.keep_cache_tokens_(on, table.cuda(), kept.cuda(), lens.cuda(), start.cuda())
    for got, c in zip(on, caches):
        assert torch.equal(got.cpu().view(torch.uint8), M.keep_tokens(c, table, kept, lens, start).view(torch.uint8))


# (a wavefront takes caches in turn from 4096 wavefronts on, on 256 CUs: two, three, eight, six and five of them here, and fewer in most last groups)
@pytest.mark.parametrize("users, heads, caches, d", [(40, 8, 19, 128), (40, 8, 20, 128), (32, 8, 67, 128), (64, 4, 25, 256), (40, 16, 19, 64)])
@pytest.mark.parametrize("most", [6, 32])
def test_few_rows_in_many_caches(users, heads, caches, d, most):
    g = torch.Generator().manual_seed(caches + most)
    bs, tokens = 4, 40
    width = tokens // bs
    table = torch.randperm(users * width + 2, generator=g)[: users * width].view(users, width).int()
    counts = [(5 * u) % (most + 1) for u in range(users)]
    counts[1] = most
    _kept(g, [_noise(g, users * width + 2, heads, bs, d) for _ in range(caches)], table, counts, tokens, [u % 9 for u in range(users)], most)


# (whole rows per workgroup, or 256 bytes of longer ones, from one workgroup per CU on: batches of 128 rows)
@pytest.mark.parametrize("users, heads, caches, d", [(4, 8, 9, 128), (4, 8, 5, 256), (5, 8, 7, 128)])
@pytest.mark.parametrize("counts", [(300, 129, 128, 1, 257), (640, 0, 127, 385, 512)])
def test_many_rows_in_many_caches(users, heads, caches, d, counts):
    g = torch.Generator().manual_seed(users + d)
    bs, tokens = 16, 700
    width = -(-tokens // bs)
    table = torch.randperm(users * width + 2, generator=g)[: users * width].view(users, width).int()
    counts, first = list(counts[:users]), [0, 3, 500, 17, 100][:users]
    _kept(g, [_noise(g, users * width + 2, heads, bs, d) for _ in range(caches)], table, counts, tokens, first, max(counts))


@pytest.mark.parametrize("counts, most", [((7, 20, 0), 20), ((90, 33, 1), 90)])
def test_more_caches_than_a_launch_takes(counts, most):
    g = torch.Generator().manual_seed(most)
    table = torch.randperm(3 * 8 + 1, generator=g)[: 3 * 8].view(3, 8).int()
    _kept(g, [_noise(g, 25, 2, 16, 64) for _ in range(200)], table, list(counts), 128, [0, 5, 64], most)


@pytest.mark.parametrize("pairs", [251, 250, 128])
@pytest.mark.parametrize("layers, block", [(24, (8, 32, 128)), (12, (8, 64, 128))])
def test_several_trips_through_the_pairs(layers, block, pairs):
    """Disjoint pairs, some of them with ids outside, of caches whose slices leave each workgroup several runs of pairs, and the scales that go with them."""
    g = torch.Generator(device="cuda").manual_seed(pairs)
    nb = 2 * pairs + 11
    caches = [torch.randint(0, 1 << 31, (nb, block[0] * block[1] * block[2] // 2), generator=g, device="cuda", dtype=torch.int32) for _ in range(layers)]
    caches += [torch.rand(nb, block[0], generator=g, device="cuda") for _ in range(layers)]
    order = torch.randperm(nb, generator=g, device="cuda").int()
    source, target = order[:pairs].clone(), order[pairs : 2 * pairs].clone()
    source[5], target[77], source[pairs - 1] = -1, nb, 1 << 30
    live = torch.ones(pairs, dtype=torch.bool, device="cuda")
    live[[5, 77, pairs - 1]] = False
    want = []
    for c in caches:
        w = c.clone()
        w[target[live].long()] = c[source[live].long()]
        want.append(w)
    torch.ops.tt.copy_cache_blocks_(caches, source, target)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
