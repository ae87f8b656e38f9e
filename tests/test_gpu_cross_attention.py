"""Attention to an encoder's states in a paged cache (``tt::paged_cross_attention``) against softmax in 64 bits.

Tolerance: a weight is rounded to bfloat16 (2^-8 of it), the same rounded weights make the normaliser, the result is rounded once more; scores are
exact products summed in float32 (at most 256 roundings of sums of 11 at these sizes, 1.7e-4 of a weight, twice with the normaliser, and the exponential's
own): 2^-8 |out| + (2 * 2^-8 * 1.005 + 6e-4) sum p |v|."""

import pytest
import torch

import __graft_entry__ as entry
import media_reference as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


@pytest.fixture(params=["rows", "planned", "stream", None], autouse=True)
def form(request, monkeypatch):
    """The forms for few rows, their parts by the longest user or by all users' lengths, the streaming loop, and what the library chooses."""
    if request.param:
        monkeypatch.setenv("TTPA_CROSS_FORM", request.param)
    return request.param


def _check(out, q, k, v, table, lens, scale, room=None, gain=1):
    """gain: scores are that much larger, and their roundings."""
    want, spread = M.cross(q, k, v, table, lens, scale, room)
    err = (out.cpu().double() - want).abs()
    tol = 2.0**-8 * want.abs() + (2 * 2.0**-8 * 1.005 + gain * 6e-4) * spread + 1e-30
    bad = ~(err <= tol)
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), float((err / tol).nan_to_num(1e9).max()))


def _inputs(g, users, hkv, grp, s, d, bs, lens, width, spare=2):
    nb = users * width + spare
    k, v = (torch.randn(nb, hkv, bs, d, generator=g).to(torch.bfloat16) for _ in range(2))
    table = (torch.randperm(nb - 1, generator=g)[: users * width] + 1).view(users, width).int()
    q = torch.randn(users, s, hkv * grp, d, generator=g).to(torch.bfloat16).transpose(1, 2)
    # what is behind the last key is anything
    for u, n in enumerate(lens):
        for c in range(width):
            if n < c * bs + bs:
                k[int(table[u, c]), :, max(0, n - c * bs) :] = float("nan")
                v[int(table[u, c]), :, max(0, n - c * bs) :] = float("nan") if c % 2 else float("inf")
    return q, k, v, table


def _run(q, k, v, table, lens, **kw):
    return torch.ops.tt.paged_cross_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.as_tensor(lens).cuda(), **kw)


@pytest.mark.parametrize("d, bs", [(64, 32), (64, 64), (128, 32), (128, 96), (128, 128), (256, 32), (256, 64)])
@pytest.mark.parametrize("hkv, grp, s", [(2, 4, 1), (2, 1, 1), (1, 16, 1), (2, 4, 5), (1, 5, 7), (1, 40, 1), (2, 2, 33), (1, 4, 96), (1, 1, 300), (2, 8, 40)])
@pytest.mark.parametrize("lens", [(0, 1, 31, 32, 33, 64), (200, 0, 127, 65), (500,)])
@pytest.mark.parametrize("known", [False, True])
def test_lengths(d, bs, hkv, grp, s, lens, known):
    g = torch.Generator().manual_seed(d + bs + s + grp)
    width = -(-max(lens) // bs) + (0 if known else 1)
    q, k, v, table = _inputs(g, len(lens), hkv, grp, s, d, bs, lens, width)
    on = [q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()]
    kw = {"most_keys": max(lens)} if known else {}
    out = torch.ops.tt.paged_cross_attention(*on, **kw)
    assert out.stride() == q.stride()
    _check(out, q, k, v, table, lens, d**-0.5)
    into = torch.full((len(lens), hkv * grp, s, d), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.ops.tt.paged_cross_attention_out(*on[:4], on[4].long(), into, **kw)
    assert torch.equal(into, out)


@pytest.mark.parametrize("d, hkv, grp, s, lens", [(64, 2, 1, 1, (9000, 17)), (128, 2, 4, 1, (6404, 5000, 1)), (128, 8, 8, 5, (4096, 513)), (256, 2, 2, 3, (3100, 40)),
                                                  (64, 4, 1, 447, (1500, 1499)), (128, 2, 4, 257, (1601, 0, 2500)), (256, 1, 2, 130, (700, 1301)),
                                                  (128, 8, 5, 65, (900, 30)), (64, 8, 1, 40, (2100,)), (128, 1, 4, 64, (7000,)), (256, 2, 4, 33, (4100, 64))])
def test_long(d, hkv, grp, s, lens):
    """Keys in parts, blocks of rows, both together."""
    g = torch.Generator().manual_seed(s + d)
    for bs in (32, 64):
        q, k, v, table = _inputs(g, len(lens), hkv, grp, s, d, bs, lens, -(-max(lens) // bs) + 3)
        for kw in ({}, {"most_keys": max(lens), "scale": 0.3}):
            _check(_run(q, k, v, table, lens, **kw), q, k, v, table, lens, kw.get("scale", d**-0.5))


@pytest.mark.parametrize("d, hq, hkv, s", [(128, 8, 2, 1), (128, 16, 2, 8), (64, 6, 3, 2), (256, 4, 2, 3), (64, 8, 1, 20)])
@pytest.mark.parametrize("users", [64, 150])
def test_many_users_of_all_lengths(d, hq, hkv, s, users):
    """One long user among short ones and none, more users than a wavefront has lanes, lengths in 64 bits: every unit of the plan once."""
    g = torch.Generator().manual_seed(users + d)
    lens = torch.randint(0, 70, (users,), generator=g)
    lens[users // 2], lens[0] = 3000, 0
    q, k, v, table = _inputs(g, users, hkv, hq // hkv, s, d, 32, lens.tolist(), 94)
    _check(_run(q, k, v, table, lens), q, k, v, table, lens, d**-0.5)


def test_lengths_beyond_the_table_and_below_zero_and_pages_outside():
    g = torch.Generator().manual_seed(1)
    q, k, v, table = _inputs(g, 4, 2, 4, 3, 128, 32, (96,) * 4, 3)
    table[1, 1], table[2, 0] = -1, k.shape[0] + 7  # read block 0
    lens = torch.tensor([1 << 40, 96, 70, -5])
    _check(_run(q, k, v, table, lens), q, k, v, table, lens, 128**-0.5)
    for tokens in (40, 200):
        q = torch.randn(4, tokens, 8, 128, generator=g).to(torch.bfloat16).transpose(1, 2)
        _check(_run(q, k, v, table, lens), q, k, v, table, lens, 128**-0.5)


@pytest.mark.parametrize("s", [1, 4, 70, 300])
def test_a_bound_below_a_length_ends_the_table(s):
    """most_keys is a promise; where it is not kept, the table ends with the block of the last promised key, in every form."""
    g = torch.Generator().manual_seed(s)
    lens = (300, 100, 0)
    q, k, v, table = _inputs(g, 3, 2, 4, s, 128, 64, lens, 5)
    out = _run(q, k, v, table, lens, most_keys=130)
    _check(out, q, k, v, table, lens, 128**-0.5, room=192)


@pytest.mark.parametrize("s", [1, 6, 50, 256])
def test_large_scores_and_infinite_values(s):
    """Scores of hundreds: one key has all the weight.  An infinite value that is attended is the result; a NaN among the attended keys is the row's."""
    g = torch.Generator().manual_seed(s)
    lens = (257, 64)
    q, k, v, table = _inputs(g, 2, 1, 4, s, 64, 32, lens, 9)
    q = (q.float() * 30).to(torch.bfloat16)
    _check(_run(q, k, v, table, lens), q, k, v, table, lens, 64**-0.5, gain=30)
    k2, v2 = k.clone(), v.clone()
    v2[int(table[0, 0]), :, 3, 5] = float("inf")
    k2[int(table[1, 1]), :, 0, 0] = float("nan")
    out = _run((q.float() / 100).to(torch.bfloat16), k2, v2, table, lens).cpu()
    assert bool((out[0, :, :, 5] == float("inf")).all()) and bool(torch.isfinite(out[0, :, :, :5]).all())
    assert bool(torch.isnan(out[1]).all())


@pytest.mark.parametrize("s", [1, 48])
def test_operands_by_strides(s):
    """Queries in head-major and token-major order, every second head, rows that vector loads cannot take; outputs in other orders."""
    g = torch.Generator().manual_seed(s)
    lens = (77, 130)
    q, k, v, table = _inputs(g, 2, 2, 4, s, 64, 32, lens, 5)
    on = [k.cuda(), v.cuda(), torch.cat([table, table], 1).cuda()[:, :5], torch.tensor(lens).cuda()]
    want = torch.ops.tt.paged_cross_attention(q.cuda().contiguous(), *on)
    _check(want, q, k, v, table, lens, 64**-0.5)
    wide = torch.zeros(2, s, 16, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, :, ::2] = q.cuda().transpose(1, 2)
    assert torch.equal(torch.ops.tt.paged_cross_attention(wide[:, :, ::2].transpose(1, 2), *on), want)
    odd = torch.zeros(2 * s * 8 * 65 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 8, s, 65)[..., :64]
    odd.copy_(q)
    assert torch.equal(torch.ops.tt.paged_cross_attention(odd, *on), want)
    for out in (torch.zeros(s, 2, 8, 64, dtype=torch.bfloat16, device="cuda").permute(1, 2, 0, 3),
                torch.zeros(2, 8, s, 67, dtype=torch.bfloat16, device="cuda")[..., 3:]):
        torch.ops.tt.paged_cross_attention_out(q.cuda(), *on, out)
        assert torch.equal(out, want)
    own = q.cuda().clone(memory_format=torch.preserve_format)
    torch.ops.tt.paged_cross_attention_out(own, *on, own)  # in the query's place
    assert torch.equal(own, want)


def test_caches_beyond_four_gibibytes():
    g = torch.Generator().manual_seed(3)
    nb, hkv, bs, d = 20000, 8, 128, 128
    k, v = (torch.zeros(nb, hkv, bs, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[19999, 3, 16384, 12000], [19998, 2, 8192, 1]], dtype=torch.int32)
    some = table.flatten().long()
    small = [torch.randn(8, hkv, bs, d, generator=g).to(torch.bfloat16) for _ in range(2)]
    for cache, x in zip((k, v), small):
        cache[some.cuda()] = x.cuda()
    lens = (500, 400)
    local = torch.arange(8).view(2, 4).int()
    for s in (1, 300):
        q = torch.randn(2, 16, s, d, generator=g).to(torch.bfloat16)
        out = torch.ops.tt.paged_cross_attention(q.cuda(), k, v, table.cuda(), torch.tensor(lens).cuda())
        _check(out, q, *small, local, lens, d**-0.5)


def test_nobody_and_no_tokens():
    k = torch.zeros(4, 2, 32, 64, dtype=torch.bfloat16, device="cuda")
    op, i = torch.ops.tt.paged_cross_attention, dict(dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 3, 64, dtype=torch.bfloat16, device="cuda")
    assert op(q, k, k, torch.zeros(0, 2, **i), torch.zeros(0, **i)).shape == q.shape
    q = torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16, device="cuda")
    assert op(q, k, k, torch.zeros(2, 2, **i), torch.zeros(2, **i)).shape == q.shape
    for s in (1, 64):  # no user has a key
        q = torch.full((3, 4, s, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
        assert bool((op(q, k, k, torch.zeros(3, 2, **i), torch.zeros(3, **i)) == 0).all())


def test_refusals():
    k = torch.zeros(4, 2, 32, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    op = torch.ops.tt.paged_cross_attention
    for args in [(q.float(), k, k, table, lens), (q[0], k, k, table, lens), (q[:, :3], k, k, table, lens), (q, k.float(), k, table, lens), (q, k, k[:2], table, lens),
                 (q, k.transpose(0, 1), k.transpose(0, 1), table, lens), (q, k, k, table.expand(2, -1), lens), (q, k, k, table, lens.expand(2)),
                 (q, k, k, table, lens.float()), (q, k, k, table.float(), lens), (q, k, k, table[:, :0], lens), (q, k, k, table, lens, -1.0),
                 (q, k, k, table, lens, 0.0), (q, k, k, table, lens, None, -1)]:
        with pytest.raises(ValueError):
            op(*args)
    small = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="multiple of 32"):
        op(q, small, small, table, lens)
    odd = torch.zeros(4, 2, 32, 96, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="head_size"):
        op(torch.zeros(1, 4, 8, 96, dtype=torch.bfloat16, device="cuda"), odd, odd, table, lens)
    for bad in [(q.clone().requires_grad_(), k, k, table, lens), (q, k.cpu(), k, table, lens), (q, k, k, table, lens.cpu())]:
        with pytest.raises(NotImplementedError):
            op(*bad)
    with pytest.raises(ValueError):
        torch.ops.tt.paged_cross_attention_out(q, k, k, table, lens, q[:, :, :4])
    with pytest.raises(ValueError, match="expanded"):
        torch.ops.tt.paged_cross_attention_out(q, k, k, table, lens, q[:, :1].clone().expand(-1, 4, -1, -1))


@pytest.mark.parametrize("s", [1, 5, 200])
def test_captured_and_on_two_streams(s):
    """A graph replayed with other lengths, pages and queries against eager calls; two streams at once."""
    g = torch.Generator().manual_seed(s)
    lens = (700, 1, 330)
    q, k, v, table = _inputs(g, 3, 2, 4, s, 128, 32, (736,) * 3, 23)
    q, k, v, table = q.cuda(), k.cuda(), v.cuda(), table.cuda()
    at = torch.tensor(lens, device="cuda")
    run = lambda: torch.ops.tt.paged_cross_attention(q, k, v, table, at)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for n in ((700, 1, 330), (0, 736, 32), (64, 65, 0), (5, 9, 600)):
        at.copy_(torch.tensor(n))
        q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16))
        table.copy_(table.flip(1))
        graph.replay()
        want = run()
        assert torch.equal(out, want)
        _check(out, q.cpu(), k.cpu(), v.cpu(), table.cpu(), n, 128**-0.5)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = [torch.ops.tt.paged_cross_attention(q, k, v, table, at) for _ in range(4)]
    here = [run() for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in other + here)
