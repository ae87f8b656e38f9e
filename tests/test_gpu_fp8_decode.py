"""Decode attention over the 8-bit cache (``tt::paged_fp8_attention_decode`` and its sparse form) against softmax in 64 bits over the
values that the cache stands for.

Tolerance.  Elements and queries enter the products exactly.  A weight is rounded to bfloat16, 2^-8 of it, and the normaliser sums the
rounded weights, so a result moves by at most 2^-8 sum p |v| / (1 - 2^-8) from the weights' and as much from the normaliser's rounding, and
it is rounded to bfloat16 itself, 2^-8 of it.  The scores are float32 sums of 64 ... 256 products: 2^-24 sqrt-free, 256 * 2^-24 of sum |q k| scale,
which is below 40 for these inputs, 6e-4 of a weight at the very most, and the hardware's exp2 adds 2^-22.
So: 2^-8 |out| + (2 * 2^-8 * 1.005 + 6e-4) sum p |v|."""

import math
import os

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _cache(nb, hkv, bs, d, g, spread=3):
    """K and V caches whose blocks have scales of their own, far apart for V; (elements, scales) twice."""
    out = []
    for i in range(2):
        x = torch.randn(nb, hkv, bs, d, generator=g)
        if i == 0:
            x[..., torch.randint(0, d, (max(1, d // 50),), generator=g)] *= 3  # channels that stand out
        x = x * 2.0 ** torch.randint(-spread * i, spread * i + 1, (nb, hkv, 1, 1), generator=g)
        s = R.scale_for(x.double())
        out.append((R.nearest_e4m3(x.double() / s[..., None, None]).float().to(torch.float8_e4m3fn), s.float()))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def _void(cache, table, lengths, lows, keep_blocks=()):
    """What nobody attends becomes NaN elements (and NaN scales where a block has no attended row)."""
    k, v, ks, vs = (t.clone() for t in cache)
    nb, _, bs, _ = k.shape
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for u, (n, lo) in enumerate(zip(lengths, lows)):
        for p in range(lo, n):
            c = p // bs
            b = int(table[u, c]) if c < table.shape[1] else 0
            used[b if 0 <= b < nb else 0, p % bs] = True
    for b in keep_blocks:
        used[b] = True
    for e in (k, v):
        e.view(torch.uint8)[~used[:, None, :, None].expand_as(e)] = 0x7F
    for s in (ks, vs):
        s[~used.any(1)] = math.nan
    return k, v, ks, vs


def _check(out, q, cache, table, cur, scale, window=0, sink=None, columns=None):
    """out, q [users, hq, d]"""
    k, v, ks, vs = cache
    users, hq, d = q.shape
    nb, hkv, bs, _ = k.shape
    grp = hq // hkv
    cap = table.shape[1] * bs
    for u in range(users):
        n = min(int(cur[u]) + 1, cap)
        if n <= 0:
            assert torch.isnan(out[u]).all()
            continue
        lo = max(0, n - window) if window else 0
        for h in range(hkv):
            cols = list(range(-(-n // bs))) if columns is None else columns[u][h]
            at = (torch.tensor(cols)[:, None] * bs + torch.arange(bs)).flatten()
            ids = [int(table[u, c]) for c in cols]
            K, V = R.gather(k, ks, ids, h), R.gather(v, vs, ids, h)
            allowed = ((at < n) & (at >= lo))[None, :].expand(grp, -1)
            rows = q[u, h * grp : h * grp + grp]
            K = torch.where(allowed[:1].T, K, torch.zeros_like(K))
            want, size = R.softmax_rows(rows, K, V, allowed, scale, None if sink is None else sink[h * grp : h * grp + grp])
            err = (out[u, h * grp : h * grp + grp].double() - want).abs()
            tol = 2.0**-8 * want.abs() + (2 * 2.0**-8 * 1.005 + 6e-4) * size + 1e-30
            assert bool((err <= tol).all()), (u, h, float((err / tol).max()))


def _setup(users, hkv, g_, d, bs, lengths, seed, extra=2):
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-n // bs)) for n in lengths]
    width = max(need) + 1
    nb = sum(need) + extra
    cache = _cache(nb, hkv, bs, d, g)
    order = torch.randperm(nb - 1, generator=g) + 1
    table = torch.full((users, width), -1, dtype=torch.int32)
    at = 0
    for u, n in enumerate(need):
        table[u, :n] = order[at : at + n].int()
        at += n
    cur = torch.tensor(lengths, dtype=torch.int32) - 1
    q = torch.randn(users, hkv * g_, d, generator=g).to(torch.bfloat16)
    return cache, table, cur, q, g


def _run(q, cache, table, cur, **kw):
    on = [t.cuda() for t in cache]
    return torch.ops.tt.paged_fp8_attention_decode(q.cuda()[None], *on, table.cuda(), cur.cuda(), **kw)[0].cpu()


@pytest.mark.parametrize("d, bs", [(64, 16), (64, 32), (128, 16), (128, 32), (128, 48), (128, 64), (128, 256), (256, 16), (256, 64)])
@pytest.mark.parametrize("hkv, grp", [(1, 1), (2, 4), (8, 1), (3, 5), (2, 16), (1, 7)])
@pytest.mark.parametrize("form", ["ranges", "few", "direct", None])
def test_lengths(d, bs, hkv, grp, form, monkeypatch):
    """From one token on, ends inside and at the ends of tiles and blocks, a padded row; whatever stands behind the last token."""
    lengths = [1, 2, 15, 16, 17, bs, bs + 1, 63, 64, 65, 0, 128, 129, 300, 2 * bs - 1]
    cache, table, cur, q, g = _setup(len(lengths), hkv, grp, d, bs, lengths, d + bs + hkv)
    cache = _void(cache, table, lengths, [0] * len(lengths))
    if form == "few":  # few wavefronts: ranges of several segments
        monkeypatch.setenv("TTPA_DECODE_WAVES_PER_CU", "0.05")
    elif form:
        monkeypatch.setenv("TTPA_DECODE_KERNEL", form)
    out = _run(q, cache, table, cur)
    _check(out, q, cache, table, cur, d**-0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("form", ["ranges", "few", "direct"])
def test_windows_and_sinks(d, form, monkeypatch):
    bs, hkv, grp = 32, 2, 4
    lengths = [1, 40, 64, 100, 257, 330, 700, 0]
    cache, table, cur, q, g = _setup(len(lengths), hkv, grp, d, bs, lengths, d)
    sink = torch.randn(hkv * grp, generator=g) * 2
    if form == "few":
        monkeypatch.setenv("TTPA_DECODE_WAVES_PER_CU", "0.03")
    else:
        monkeypatch.setenv("TTPA_DECODE_KERNEL", form)
    for window in (1, 7, 64, 100, 300, 100000):
        lows = [max(0, n - window) for n in lengths]
        void = _void(cache, table, lengths, lows)
        out = _run(q, void, table, cur.long(), sliding_window_size=window, attention_sink=sink.cuda(), scale=0.3)
        _check(out, q, void, table, cur, 0.3, window, sink)
    out = _run(q, cache, table, cur, scale=-0.1)
    _check(out, q, cache, table, cur, -0.1)


def test_long_ragged_contexts_default_choice():
    d, bs, hkv, grp = 128, 64, 4, 8
    lengths = [5000, 1, 20000, 333, 0, 12000, 64, 4097, 3000, 9000, 2, 700]
    cache, table, cur, q, g = _setup(len(lengths), hkv, grp, d, bs, lengths, 3)
    out = _run(q, cache, table, cur)
    _check(out, q, cache, table, cur, d**-0.5)


@pytest.mark.parametrize("users, tokens", [(24, 2304), (24, 1000), (70, 800), (70, 300)])
def test_long_and_short_lists_at_head_size_64_on_wide_tables(users, tokens):
    """Tables wide enough for the larger grid; lists that use all of it, and lists that leave half of it empty."""
    lengths = [max(0, tokens - 37 * (u % 9)) for u in range(users)]
    lengths[3], lengths[5] = 0, 1
    cache, table, cur, q, _ = _setup(users, 8, 2, 64, 64, lengths, users + tokens)
    wide = torch.full((users, 80), -1, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    cache = _void(cache, wide, lengths, [0] * users)
    out = _run(q, cache, wide, cur)
    _check(out, q, cache, wide, cur, 64**-0.5)


def test_more_users_than_a_wavefront_has_lanes_and_positions_beyond_the_table():
    d, bs, hkv, grp, users = 64, 32, 2, 2, 150
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 200, (users,), generator=g).tolist()
    cache, table, cur, q, g = _setup(users, hkv, grp, d, bs, lengths, 4)
    cur[3] = 10**6  # all that the table has; its free columns read block 0, as ids outside the cache do
    table[5, 0] = 10**6
    for form in (None, "ranges"):
        if form:
            os.environ["TTPA_DECODE_KERNEL"] = form
        try:
            out = _run(q, cache, table, cur)
        finally:
            os.environ.pop("TTPA_DECODE_KERNEL", None)
        _check(out, q, cache, table, cur, d**-0.5)


def test_blocks_whose_scales_are_far_apart():
    """One block's values are 2^40 times the others': neither it nor they lose bits."""
    d, bs, hkv, grp = 128, 32, 1, 4
    lengths = [200]
    cache, table, cur, q, g = _setup(1, hkv, grp, d, bs, lengths, 8)
    k, v, ks, vs = cache
    for at, e in ((0, 40), (3, -60), (5, 100)):
        vs2 = vs.clone()
        vs2[int(table[0, at])] *= 2.0**e
        out = _run(q, (k, v, ks, vs2), table, cur)
        _check(out, q, (k, v, ks, vs2), table, cur, d**-0.5)
    # and a key block that takes all of the weight, or none
    for e in (6, -100):
        ks2 = ks.clone()
        ks2[int(table[0, 2])] *= 2.0**e
        out = _run(q, (k, v, ks2, vs), table, cur, scale=0.02)
        _check(out, q, (k, v, ks2, vs), table, cur, 0.02)


def test_a_nan_that_is_attended_is_seen():
    d, bs, hkv, grp = 128, 32, 2, 4
    cache, table, cur, q, g = _setup(2, hkv, grp, d, bs, [100, 100], 8)
    k, v, ks, vs = (t.clone() for t in cache)
    k.view(torch.uint8)[int(table[0, 1]), 0, 5, 7] = 0x7F
    v.view(torch.uint8)[int(table[1, 2]), 1, 5, 7] = 0x7F
    out = _run(q, (k, v, ks, vs), table, cur)
    assert torch.isnan(out[0, :4]).all() and not torch.isnan(out[0, 4:]).any()
    assert torch.isnan(out[1, 4:, 7]).all() and int(torch.isnan(out[1]).sum()) == 4


def test_strided_operands_and_outputs():
    d, bs, hkv, grp = 128, 32, 2, 4
    cache, table, cur, q, g = _setup(5, hkv, grp, d, bs, [100, 3, 64, 200, 31], 8)
    on = [t.cuda() for t in cache]
    want = torch.ops.tt.paged_fp8_attention_decode(q.cuda()[None], *on, table.cuda(), cur.cuda())
    wide = torch.zeros(5, 3, hkv * grp, d, dtype=torch.bfloat16).cuda()
    wide[:, 1] = q.cuda()
    assert torch.equal(torch.ops.tt.paged_fp8_attention_decode(wide[:, 1][None], *on, table.cuda(), cur.cuda()), want)
    heads_first = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)[None]
    assert torch.equal(torch.ops.tt.paged_fp8_attention_decode(heads_first, *on, table.cuda(), cur.cuda()), want)
    odd = torch.zeros(5 * (hkv * grp * d + 1) + 3, dtype=torch.bfloat16).cuda()[3:].as_strided((1, 5, hkv * grp, d), (0, hkv * grp * d + 1, d, 1))
    torch.ops.tt.paged_fp8_attention_decode_out(q.cuda()[None], *on, table.cuda(), cur.cuda(), odd)
    assert torch.equal(odd, want)
    view = torch.zeros_like(wide)
    torch.ops.tt.paged_fp8_attention_decode_out(q.cuda()[None], *on, table.cuda(), cur.cuda(), view[:, 2][None])
    assert torch.equal(view[:, 2][None], want) and int(view[:, :2].count_nonzero()) == 0
    pages = torch.zeros(5, 2 * table.shape[1], dtype=torch.int32).cuda()
    pages[:, ::2] = table.cuda()
    assert torch.equal(torch.ops.tt.paged_fp8_attention_decode(q.cuda()[None], *on, pages[:, ::2], cur.cuda()), want)
    assert torch.equal(torch.ops.tt.paged_fp8_attention_decode(q.cuda()[None], *on, table.long().cuda(), cur.to(torch.int16).cuda()), want)
    empty = torch.ops.tt.paged_fp8_attention_decode(q[:0].cuda()[None], *on, table[:0].cuda(), cur[:0].cuda())
    assert empty.shape == (1, 0, hkv * grp, d)


def test_a_cache_beyond_four_gibibytes():
    d, bs, hkv, grp = 128, 64, 8, 2
    lengths = [150, 64]
    cache, table, cur, q, g = _setup(2, hkv, grp, d, bs, lengths, 12)
    nb = (1 << 32) // (hkv * d * bs) + 20
    few = cache[0].shape[0]
    big = []
    for e in cache[:2]:
        t = torch.empty(nb, hkv, bs, d, dtype=torch.uint8, device="cuda")
        t[nb - few :] = e.view(torch.uint8).cuda()
        big.append(t.view(torch.float8_e4m3fn))
    scales = []
    for s in cache[2:]:
        t = torch.ones(nb, hkv, device="cuda")
        t[nb - few :] = s.cuda()
        scales.append(t)
    moved = torch.where(table >= 0, table + (nb - few), table)
    small = _run(q, cache, table, cur)
    out = torch.ops.tt.paged_fp8_attention_decode(q.cuda()[None], *big, *scales, moved.cuda(), cur.cuda())[0].cpu()
    assert torch.equal(out, small)


# --------------------------------------------------------------------------- #
# sparse
# --------------------------------------------------------------------------- #
def _bounds(cache):
    k, _, ks, _ = cache
    x = R.values(k) * ks.double()[..., None, None]
    return torch.stack([x.amin(2), x.amax(2)], 2).to(torch.bfloat16)


def _sparse(q, cache, bounds, table, cur, kept, **kw):
    on = [t.cuda() for t in cache]
    out, cols = torch.ops.tt.paged_fp8_sparse_attention_decode(q.cuda()[None], *on, bounds.cuda(), table.cuda(), cur.cuda(), kept, **kw)
    return out[0].cpu(), cols.cpu()


def _check_sparse(out, cols, q, cache, bounds, table, cur, kept, scale):
    users, hq, _ = q.shape
    hkv, bs = cache[0].shape[1:3]
    grp = hq // hkv
    chosen = []
    for u in range(users):
        chosen.append([])
        n = min(int(cur[u]) + 1, table.shape[1] * bs)
        for h in range(hkv):
            want = R.choose(q[u, h * grp : h * grp + grp], bounds, table[u].tolist(), h, -(-n // bs), kept) if n > 0 else []
            assert cols[u, h].tolist() == want + [-1] * (kept - len(want)), (u, h)
            chosen[u].append(want)
    _check(out, q, cache, table, cur, scale, columns=chosen)


@pytest.mark.parametrize("d, bs", [(64, 16), (64, 64), (128, 32), (128, 64), (256, 32)])
@pytest.mark.parametrize("hkv, grp", [(1, 1), (2, 2), (8, 4), (2, 5), (2, 8), (1, 16)])
@pytest.mark.parametrize("kept", [2, 3, 9, 40])
def test_sparse(d, bs, hkv, grp, kept):
    lengths = [1, bs, bs + 1, 5 * bs, 12 * bs + 3, 0, 45 * bs - 1, 8 * bs + 1, 9 * bs]
    cache, table, cur, q, g = _setup(len(lengths), hkv, grp, d, bs, lengths, d + hkv + kept)
    bounds = _bounds(cache)
    out, cols = _sparse(q, cache, bounds, table, cur, kept)
    _check_sparse(out, cols, q, cache, bounds, table, cur, kept, d**-0.5)


def test_sparse_long_contexts():
    d, bs, hkv, grp = 64, 16, 2, 4
    lengths = [16 * 5000, 16 * 4096 + 7, 16 * 1025]
    cache, table, cur, q, g = _setup(len(lengths), hkv, grp, d, bs, lengths, 6)
    bounds = _bounds(cache)
    for kept in (16, 700):
        out, cols = _sparse(q, cache, bounds, table, cur, kept, scale=0.05)
        _check_sparse(out, cols, q, cache, bounds, table, cur, kept, 0.05)


@pytest.mark.parametrize("blocks", [30, 600, 5000])
def test_sparse_ties_and_bounds_that_are_no_numbers(blocks):
    """Equal scores: the lower columns.  Bounds of infinity or NaN: kept ahead of all numbers.  A table that names one block again and again."""
    d, bs, hkv, grp = 64, 16, 2, 4
    g = torch.Generator().manual_seed(blocks)
    nb = 40
    cache = _cache(nb, hkv, bs, d, g, 1)
    bounds = _bounds(cache)
    bounds[7, :, 1, 3], bounds[9, 0, 0, 5], bounds[11, 1, :, :] = math.inf, math.nan, 0.0
    table = torch.randint(0, nb, (3, blocks), generator=g).int()
    table[1] = 5
    table[2] = torch.where(table[2] % 2 == 0, 11, 12)
    cur = torch.tensor([blocks * bs - 1, blocks * bs - 9, blocks * bs - 16])
    q = torch.randn(3, hkv * grp, d, generator=g).to(torch.bfloat16)
    q[2, 0] = 0.0
    for kept in (2, 5, 29):
        out, cols = _sparse(q, cache, bounds, table, cur, kept)
        _check_sparse(out, cols, q, cache, bounds, table, cur, kept, d**-0.5)


def test_sparse_more_segments_than_one_pass_takes():
    d, bs, hkv, grp, users = 64, 16, 8, 1, 300
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(1, 100, (users,), generator=g).tolist()
    cache, table, cur, q, g = _setup(users, hkv, grp, d, bs, lengths, 2)
    bounds = _bounds(cache)
    out, cols = _sparse(q, cache, bounds, table, cur.long(), 3)
    _check_sparse(out, cols, q, cache, bounds, table, cur, 3, d**-0.5)


@pytest.mark.parametrize("d, width", [(64, 400), (128, 2500), (256, 1300)])
def test_sparse_many_contexts_of_many_blocks_on_wide_tables(d, width):
    """A workgroup scores several parts of a context; tables that go on behind the contexts."""
    bs, hkv, grp, nb, users = 16, 8, 2, 60, 150
    g = torch.Generator().manual_seed(d)
    cache = _cache(nb, hkv, bs, d, g)
    bounds = _bounds(cache)
    table = torch.randint(0, nb, (users, width), generator=g).int()
    cur = torch.randint(-1, 300 * bs, (users,), generator=g)
    q = torch.randn(users, hkv * grp, d, generator=g).to(torch.bfloat16)
    out, cols = _sparse(q, cache, bounds, table, cur, 7, scale=0.05)
    _check_sparse(out, cols, q, cache, bounds, table, cur, 7, 0.05)


@pytest.mark.parametrize("d, blocks", [(64, 8300), (128, 9001)])
def test_sparse_tables_beyond_what_is_held(d, blocks):
    """More columns than scores and pages are kept on the chip for, short contexts among the long ones."""
    bs, hkv, grp, nb = 16, 1, 4, 300
    g = torch.Generator().manual_seed(blocks)
    cache = _cache(nb, hkv, bs, d, g)
    bounds = _bounds(cache)
    table = torch.randint(0, nb, (4, blocks), generator=g).int()
    table[0, 5000:6000] = 17  # (ties across the last place)
    cur = torch.tensor([blocks * bs - 3, 40 * bs, 3, -1])
    q = torch.randn(4, hkv * grp, d, generator=g).to(torch.bfloat16)
    for kept in (2, 33, 600):
        out, cols = _sparse(q, cache, bounds, table, cur, kept, scale=0.05)
        _check_sparse(out, cols, q, cache, bounds, table, cur, kept, 0.05)


def test_sparse_strides():
    d, bs, hkv, grp = 128, 32, 2, 4
    cache, table, cur, q, g = _setup(4, hkv, grp, d, bs, [300, 3, 64, 200], 8)
    bounds = _bounds(cache)
    on = [t.cuda() for t in cache]
    args = (*on, bounds.cuda(), table.cuda(), cur.cuda())
    want, cols = torch.ops.tt.paged_fp8_sparse_attention_decode(q.cuda()[None], *args, 4)
    wide = torch.zeros(4, 2, hkv * grp, d, dtype=torch.bfloat16).cuda()
    wide[:, 1] = q.cuda()
    out = torch.zeros_like(wide)
    got = torch.ops.tt.paged_fp8_sparse_attention_decode_out(wide[:, 1][None], *args, out[:, 0][None], 4)
    assert torch.equal(out[:, 0][None], want) and torch.equal(got, cols) and int(out[:, 1].count_nonzero()) == 0


def test_refusals():
    cache, table, cur, q, _ = _setup(2, 2, 4, 64, 32, [40, 20], 1)
    bounds = _bounds(cache).cuda()
    k, v, ks, vs = (t.cuda() for t in cache)
    q, table, cur = q.cuda()[None], table.cuda(), cur.cuda()
    op, sparse = torch.ops.tt.paged_fp8_attention_decode, torch.ops.tt.paged_fp8_sparse_attention_decode
    for args in [(q.float(), k, v, ks, vs, table, cur), (q[0], k, v, ks, vs, table, cur), (q, k, v[:1], ks, vs, table, cur),
                 (q, k, v, ks, vs[:, :1], table, cur), (q, k, v, ks, vs, table[:1], cur), (q, k, v, ks, vs, table, cur[:1]),
                 (q[:, :, :3], k, v, ks, vs, table, cur), (q, k, v, ks, vs, table, cur.float()), (q, k.view(torch.uint8), v, ks, vs, table, cur),
                 (q, k, v, ks, vs, table, cur, torch.zeros(3).cuda()), (q, k, v, ks, vs, table, cur, None, None, 0)]:
        with pytest.raises(ValueError):
            op(*args)
    wide = torch.zeros(1, 2, 34, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="up to 16"):
        op(wide, k, v, ks, vs, table, cur)
    for args in [(q, k, v, ks, vs, bounds.float(), table, cur, 4), (q, k, v, ks, vs, bounds[:1], table, cur, 4), (q, k, v, ks, vs, bounds, table, cur, 1)]:
        with pytest.raises(ValueError):
            sparse(*args)
    with pytest.raises(ValueError):
        torch.ops.tt.paged_fp8_attention_decode_out(q, k, v, ks, vs, table, cur, torch.empty_like(q)[:, :1])
    with pytest.raises(NotImplementedError):
        op(q.clone().requires_grad_(), k, v, ks, vs, table, cur)


def test_expanded_outputs_are_refused():
    cache, table, cur, q, _ = _setup(2, 2, 2, 64, 32, [40, 50], 1)
    on, out = [t.cuda() for t in cache], torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device="cuda").expand(-1, 2, -1, -1)
    with pytest.raises(ValueError, match="expanded"):
        torch.ops.tt.paged_fp8_attention_decode_out(q.cuda()[None], *on, table.cuda(), cur.cuda(), out)
    with pytest.raises(ValueError, match="expanded"):
        torch.ops.tt.paged_fp8_sparse_attention_decode_out(q.cuda()[None], *on, _bounds(cache).cuda(), table.cuda(), cur.cuda(), out, 2)
    into = torch.zeros(600, dtype=torch.bfloat16, device="cuda").as_strided((1, 2, 4, 64), (0, 128, 64, 1))
    with pytest.raises(ValueError, match="overlap itself"):
        torch.ops.tt.paged_fp8_attention_decode_out(q.cuda()[None], *on, table.cuda(), cur.cuda(), into)


def test_sparse_decode_and_chunks_over_a_cache_beyond_four_gibibytes():
    d, bs, hkv, grp = 128, 64, 8, 2
    lengths = [700, 64]
    cache, table, cur, q, g = _setup(2, hkv, grp, d, bs, lengths, 13)
    nb, few = (1 << 32) // (hkv * d * bs) + 20, cache[0].shape[0]

    def far(t):
        big = torch.zeros(nb, *t.shape[1:], dtype=t.dtype, device="cuda") if t.dtype != torch.float8_e4m3fn else torch.empty(
            nb, *t.shape[1:], dtype=torch.uint8, device="cuda").view(t.dtype)
        big.view(torch.uint8)[nb - few :] = t.contiguous().view(torch.uint8).cuda()
        return big

    bounds = _bounds(cache)
    moved = torch.where(table >= 0, table + (nb - few), table).cuda()
    near, there = [t.cuda() for t in (*cache, bounds)], [far(t) for t in (*cache, bounds)]
    tt, on = torch.ops.tt, q.cuda()[None]
    want = tt.paged_fp8_sparse_attention_decode(on, *near, table.cuda(), cur.cuda(), 4)
    got = tt.paged_fp8_sparse_attention_decode(on, *there, moved, cur.cuda(), 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rows = torch.randn(2, hkv * grp, 40, d, generator=g).to(torch.bfloat16).cuda()
    start = torch.tensor([20]).cuda()
    assert torch.equal(tt.chunked_fp8_attention(rows, *there[:4], moved[:, :1], start), tt.chunked_fp8_attention(rows, *near[:4], table[:, :1].cuda(), start))
