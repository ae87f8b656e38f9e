"""Attention of a prompt's chunk over the 8-bit cache (``tt::chunked_fp8_attention``) against softmax in 64 bits over the values that
the cache stands for.  Tolerance: a weight is rounded to bfloat16 (2^-8 of it) and the normaliser may be the rounded or the exact sum, the
result is rounded once more; scores as in the decode's test: 2^-8 |out| + (2 * 2^-8 * 1.005 + 6e-4) sum p |v|."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R
from test_gpu_fp8_decode import _cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _check(out, q, cache, table, start, scale):
    k, v, ks, vs = cache
    users, hq, s, d = q.shape
    hkv, bs = k.shape[1:3]
    grp = hq // hkv
    cols = min(table.shape[1], -(-(start + s) // bs))
    at = torch.arange(cols * bs)
    allowed = at[None, :] <= start + torch.arange(s)[:, None]
    for u in range(users):
        for h in range(hkv):
            ids = table[u, :cols].tolist()
            K, V = R.gather(k, ks, ids, h), R.gather(v, vs, ids, h)
            K = torch.where(allowed.any(0)[:, None], K, torch.zeros_like(K))
            for g in range(grp):
                want, size = R.softmax_rows(q[u, h * grp + g], K, V, allowed, scale)
                err = (out[u, h * grp + g].double() - want).abs()
                tol = 2.0**-8 * want.abs() + (2 * 2.0**-8 * 1.005 + 6e-4) * size + 1e-30
                assert bool((err <= tol).all()), (u, h, g, float((err / tol).max()))


@pytest.mark.parametrize("d, bs", [(64, 32), (64, 64), (128, 32), (128, 96), (128, 128), (256, 32), (256, 64)])
@pytest.mark.parametrize("users, hkv, grp, s, start", [(1, 2, 4, 32, 0), (2, 1, 1, 64, 96), (1, 8, 4, 96, 1000), (3, 2, 2, 33, 64), (1, 1, 8, 1, 130),
                                                       (1, 2, 5, 160, 64)])
@pytest.mark.parametrize("known", [False, True])
@pytest.mark.parametrize("form", ["few", "copies", None])
def test_chunks(d, bs, users, hkv, grp, s, start, known, form, monkeypatch):
    if form:
        monkeypatch.setenv("TTPA_CHUNK_FORM", form)
    g = torch.Generator().manual_seed(d + bs + s)
    width = -(-(start + s) // bs) + 2
    nb = users * width + 3
    cache = _cache(nb, hkv, bs, d, g)
    table = torch.randperm(nb, generator=g)[: users * width].view(users, width).int()
    # rows behind the chunk and blocks behind it hold anything
    k, v, ks, vs = cache
    for u in range(users):
        for c in range(width):
            first = start + s - c * bs
            if first < bs:
                for e in (k, v):
                    e.view(torch.uint8)[int(table[u, c]), :, max(first, 0) :] = 0x7F
                if first <= 0:
                    ks[int(table[u, c])] = vs[int(table[u, c])] = float("nan")
    if users > 1:
        table[1, 0] = nb + 5  # reads block 0
    q = torch.randn(users, s, hkv * grp, d, generator=g).to(torch.bfloat16).transpose(1, 2)
    args = [t.cuda() for t in (k, v, ks, vs)]
    kw = {"most_keys": start + s} if known else {}
    if users > 1:  # (block 0 may be one with rows that hold anything)
        k.view(torch.uint8)[0], v.view(torch.uint8)[0], ks[0], vs[0] = 0x31, 0x29, 0.5, 2.0
        args = [t.cuda() for t in (k, v, ks, vs)]
        table[table == 0] = nb - 1
        k.view(torch.uint8)[nb - 1], v.view(torch.uint8)[nb - 1], ks[nb - 1], vs[nb - 1] = 0x39, 0x21, 0.5, 1.0
        args = [t.cuda() for t in (k, v, ks, vs)]
    out = torch.ops.tt.chunked_fp8_attention(q.cuda(), *args, table.cuda(), torch.tensor([start]).cuda(), **kw)
    _check(out.cpu(), q, (k, v, ks, vs), table, start, d**-0.5)
    into = torch.zeros(users, s, hkv * grp, d, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    torch.ops.tt.chunked_fp8_attention_out(q.cuda(), *args, table.cuda(), torch.tensor(start, dtype=torch.int32).cuda(), into, **kw)
    assert torch.equal(into, out)


def test_a_chunk_of_many_rows_and_an_output_that_stores_cannot_take():
    d, bs, hkv, grp, s, start = 128, 64, 2, 4, 384, 2048
    g = torch.Generator().manual_seed(5)
    width = (start + s) // bs
    cache = _cache(width + 1, hkv, bs, d, g)
    table = (torch.randperm(width, generator=g) + 1)[None].int()
    q = torch.randn(1, hkv * grp, s, d, generator=g).to(torch.bfloat16)
    args = [t.cuda() for t in cache]
    odd = torch.zeros(hkv * grp * s * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(1, hkv * grp, s, d)
    torch.ops.tt.chunked_fp8_attention_out(q.cuda(), *args, table.cuda(), torch.tensor([start]).cuda(), odd)
    _check(odd.cpu(), q, cache, table, start, d**-0.5)


def test_refusals():
    g = torch.Generator().manual_seed(5)
    k, v, ks, vs = (t.cuda() for t in _cache(4, 2, 32, 64, g))
    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16, device="cuda")
    table, start = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    op = torch.ops.tt.chunked_fp8_attention
    for args in [(q.float(), k, v, ks, vs, table, start), (q[0], k, v, ks, vs, table, start), (q[:, :3], k, v, ks, vs, table, start),
                 (q, k, v, ks, vs, table.expand(2, -1), start), (q, k, v, ks, vs, table, start.expand(2)), (q, k, v, ks, vs, table, start.float()),
                 (q, k, v, ks, vs, table, start, -1.0), (q, k, v, ks, vs, table, start, None, -1), (q, k, v, ks.half(), vs, table, start)]:
        with pytest.raises(ValueError):
            op(*args)
    small = torch.zeros(4, 2, 16, 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        op(q, small, small.clone(), ks, vs, table, start)
    with pytest.raises(NotImplementedError):
        op(q.clone().requires_grad_(), k, v, ks, vs, table, start)
    assert op(q[:, :, :0], k, v, ks, vs, table, start).shape == (1, 4, 0, 64)


def test_users_in_several_passes(monkeypatch):
    """A table so wide that the copies of three users' blocks do not fit the scratch at once: two passes, of two users and of one."""
    monkeypatch.setenv("TTPA_CHUNK_FORM", "copies")
    d, bs, hkv, grp, s, start = 128, 64, 8, 2, 70, 300
    g = torch.Generator().manual_seed(9)
    cache = _cache(20, hkv, bs, d, g)
    table = torch.full((3, 11500), -1, dtype=torch.int32)
    table[:, :6] = (torch.randperm(18, generator=g) + 1).view(3, 6).int()
    q = torch.randn(3, hkv * grp, s, d, generator=g).to(torch.bfloat16)
    args = [t.cuda() for t in cache]
    op, at = torch.ops.tt.chunked_fp8_attention, torch.tensor([start]).cuda()
    out = op(q.cuda(), *args, table.cuda(), at)
    _check(out.cpu(), q, cache, table, start, d**-0.5)


@pytest.mark.parametrize("form", ["few", "copies"])
def test_captured_prompts_and_chunks(form, monkeypatch):
    """A prompt's write and a chunk over it in one graph, replayed at other starts and with other keys; every replay against the eager calls."""
    monkeypatch.setenv("TTPA_CHUNK_FORM", form)
    d, bs, hkv, grp, s = 128, 32, 2, 4, 64
    g = torch.Generator().manual_seed(10)
    state = [t.cuda() for t in _cache(40, hkv, bs, d, g)]
    table = (torch.randperm(39, generator=g) + 1)[:24].view(2, 12).int().cuda()
    fill = (torch.arange(2 * 2) + 36).view(2, 2).int().cuda()
    k, v = (torch.randn(2, hkv, s, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(2, hkv * grp, s, d, generator=g).to(torch.bfloat16).cuda()
    rows, start = torch.tensor([0, 1]).cuda(), torch.tensor([64]).cuda()
    tt = torch.ops.tt

    def run(cache):
        tt.paged_fill_fp8_cache_(*cache, k, v, fill, rows)
        return tt.chunked_fp8_attention(q, *cache, table, start)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run([t.clone() for t in state])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(state)
    for n, at in enumerate((0, 128, 32, 320, 64)):
        start.fill_(at)
        fill[:, 0] = table[:, (n + 1) % 4]
        fill[:, 1] = table[:, 10]
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).to(torch.bfloat16))
        copy = [t.clone() for t in state]
        graph.replay()
        want = run(copy)
        if n % 2:
            torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state, copy))


def test_expanded_outputs_are_refused():
    cache = [t.cuda() for t in _cache(4, 2, 32, 64, torch.Generator().manual_seed(5))]
    q = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16, device="cuda")
    table, start = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="expanded"):
        torch.ops.tt.chunked_fp8_attention_out(q, *cache, table, start, q[:1].clone().expand(2, -1, -1, -1))


@pytest.mark.parametrize("d, hq, hkv", [(64, 8, 1), (128, 16, 2), (256, 4, 4)])
@pytest.mark.parametrize("form", ["few", "copies"])
def test_chunks_that_begin_before_the_prompt_or_end_behind_the_table(d, hq, hkv, form, monkeypatch):
    """Rows in front of the prompt attend nothing; rows behind the table attend what it holds."""
    monkeypatch.setenv("TTPA_CHUNK_FORM", form)
    g = torch.Generator().manual_seed(d)
    bs, s = 32, 40
    cache = _cache(6, hkv, bs, d, g)
    table = torch.tensor([[2, 5, 1, 4]], dtype=torch.int32)
    q = torch.randn(1, hq, s, d, generator=g).to(torch.bfloat16)
    on = [t.cuda() for t in cache]
    for start in (-7, 100, 127, 400):
        out = torch.ops.tt.chunked_fp8_attention(q.cuda(), *on, table.cuda(), torch.tensor([start]).cuda()).cpu()
        if start < 0:
            assert torch.isnan(out[:, :, : -start]).all()
            _check(out[:, :, -start:], q[:, :, -start:], cache, table, 0, d**-0.5)
        else:
            _check(out, q, cache, table, start, d**-0.5)


def test_few_rows_over_many_parts_and_many_blocks_of_rows(monkeypatch):
    monkeypatch.setenv("TTPA_CHUNK_FORM", "few")
    g = torch.Generator().manual_seed(11)
    for d, hq, hkv, users, s, start in ((64, 2, 1, 1, 3, 9000), (128, 8, 4, 2, 100, 4000), (256, 6, 2, 1, 50, 5000), (128, 40, 8, 3, 7, 300)):
        bs, width = 64, -(-(start + s) // 64) + 5
        cache = _cache(width + 4, hkv, bs, d, g)
        table = torch.stack([torch.randperm(width + 4, generator=g)[:width] for _ in range(users)]).int()
        q = torch.randn(users, s, hq, d, generator=g).to(torch.bfloat16).transpose(1, 2)
        on = [t.cuda() for t in cache]
        for known in (0, start + s):
            out = torch.ops.tt.chunked_fp8_attention(q.cuda(), *on, table.cuda(), torch.tensor([start]).cuda(), most_keys=known)
            _check(out.cpu(), q, cache, table, start, d**-0.5)


@pytest.mark.parametrize("form", ["few", "copies", None])
@pytest.mark.parametrize("d, hq, hkv", [(64, 8, 2), (128, 8, 1), (256, 4, 4)])
def test_a_bound_below_the_chunk_ends_the_table(d, hq, hkv, form, monkeypatch):
    """most_keys is a promise; where it is not kept, both forms attend what the table holds up to the block of the last promised key."""
    if form:
        monkeypatch.setenv("TTPA_CHUNK_FORM", form)
    g = torch.Generator().manual_seed(d)
    bs, s, start = 32, 40, 88
    cache = _cache(9, hkv, bs, d, g)
    table = torch.tensor([[2, 5, 1, 4, 7, 3], [6, 8, 1, 2, 4, 5]], dtype=torch.int32)
    q = torch.randn(2, hq, s, d, generator=g).to(torch.bfloat16)
    on = [t.cuda() for t in cache]
    for most in (1, 32, 33, 64, 95, 96, 97, 127, 128, 129):
        out = torch.ops.tt.chunked_fp8_attention(q.cuda(), *on, table.cuda(), torch.tensor([start]).cuda(), most_keys=most).cpu()
        _check(out, q, cache, table[:, : -(-most // bs)], start, d**-0.5)
