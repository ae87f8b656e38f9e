"""The writers of the 8-bit cache (``tt::paged_update_fp8_cache_``, ``tt::qk_norm_rope_update_fp8_``, ``tt::paged_fill_fp8_cache_``) against
their definition in 64 bits: elements, scales and bounds are whole steps of exact numbers, so all of them are equal."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R

pytestmark = pytest.mark.gpu
SHAPES = [(2, 64, 32), (8, 128, 64), (3, 256, 16), (5, 128, 128)]  # KV heads, head size, block size


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _noise(nb, hkv, bs, d, seed, bounds=True):
    """A cache with anything in it: every byte, any scale of the range."""
    g = torch.Generator().manual_seed(seed)
    e = [torch.randint(0, 256, (nb, hkv, bs, d), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn).cuda() for _ in range(2)]
    s = [torch.ldexp(torch.ones(nb, hkv), torch.randint(-12, 4, (nb, hkv), generator=g)).cuda() for _ in range(2)]
    b = torch.randn(nb, hkv, 2, d, generator=g).to(torch.bfloat16).cuda() if bounds else None
    return (*e, *s), b, g


def _same(want, cache, bounds=None):
    assert want.differences(*cache, bounds) == {}


@pytest.mark.parametrize("hkv, d, bs", SHAPES)
@pytest.mark.parametrize("bounds", [False, True])
def test_tokens_one_after_another(hkv, d, bs, bounds):
    """Every position of two blocks and of the start of a third, with magnitudes that grow, shrink and vanish."""
    users, nb = 3, 16
    cache, b, g = _noise(nb, hkv, bs, d, hkv, bounds)
    table = torch.randperm(nb, generator=g)[: users * 3].view(users, 3).int()
    want = R.Cache(*cache, b)
    for p in range(2 * bs + 3):
        gain = 2.0 ** torch.randint(-9, 7, (users, 1, 1), generator=g).double() * (p % 7 != 3)
        k, v = ((torch.randn(users, hkv, d, generator=g) * gain).to(torch.bfloat16) for _ in range(2))
        pos = torch.full((users,), p, dtype=torch.int32)
        want.update(k, v, pos, table)
        torch.ops.tt.paged_update_fp8_cache_(*cache, k.cuda()[None], v.cuda()[None], pos.cuda(), table.cuda(), b)
        if p % 5 == 0 or p > 2 * bs:
            _same(want, cache, b)
    _same(want, cache, b)


def test_special_values():
    """NaN, infinities, zeros, the largest and the smallest numbers, ties of the rounding."""
    hkv, d, bs = 2, 64, 16
    rows = torch.zeros(8, hkv, d)
    rows[1, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0])
    rows[2, :, 0] = 3.3895313892515355e38
    rows[3, :, :] = -3.3895313892515355e38
    rows[4, :, 3] = 9.2e-41
    rows[5] = torch.arange(d) / 16.0 + 0.03125
    rows[6, :, 7] = 448.0
    rows[7, :, 7] = 450.0
    for first in range(8):  # whichever row begins the block
        cache, b, g = _noise(4, hkv, bs, d, first)
        want = R.Cache(*cache, b)
        table = torch.tensor([[2, 1]])
        for p in range(8):
            x = rows[(first + p) % 8].to(torch.bfloat16)[None]
            want.update(x, -x, torch.tensor([p]), table)
            torch.ops.tt.paged_update_fp8_cache_(*cache, x.cuda()[None], -x.cuda()[None], torch.tensor([p]).cuda(), table.cuda(), b)
            _same(want, cache, b)


def test_users_that_write_nothing_and_users_of_one_block():
    hkv, d, bs, users = 8, 128, 32, 200
    cache, b, g = _noise(12, hkv, bs, d, 5)
    # blocks of several users, with other rows and with the same row; padded rows, columns outside the table, blocks outside the cache
    table = torch.randint(-2, 14, (users, 3), generator=g).long()
    pos = torch.randint(-3, 4 * bs, (users,), generator=g)
    k, v = (torch.randn(users, hkv + 2, d, generator=g).to(torch.bfloat16) * 2.0 ** torch.randint(-4, 5, (users, 1, 1), generator=g) for _ in range(2))
    want = R.Cache(*cache, b)
    want.update(k[:, :hkv], v[:, :hkv], pos, table)
    torch.ops.tt.paged_update_fp8_cache_(*cache, k.to(torch.bfloat16).cuda()[None], v.to(torch.bfloat16).cuda()[None], pos.cuda(), table.cuda(), b)
    _same(want, cache, b)


@pytest.mark.parametrize("hq, hkv, d, bs, rotary", [(8, 2, 64, 32, 64), (32, 8, 128, 64, 128), (6, 3, 256, 16, 64), (64, 8, 128, 32, 128)])
@pytest.mark.parametrize("users", [1, 5, 70])
def test_the_step_in_one_launch(hq, hkv, d, bs, rotary, users):
    """Norm, rotation and write in one launch give what the operators give in turn, bit for bit."""
    from tt_xla_amd.fp8_ops import rope_table

    one, b1, g = _noise(users + 4, hkv, bs, d, users)
    two, b2 = tuple(t.clone() for t in one), b1.clone()
    qkv = torch.randn(users, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).cuda()
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
    qw, kw = (1 + torch.rand(d, generator=g).cuda() for _ in range(2))
    angles = rope_table(3 * bs, rotary, device="cuda")
    table = torch.randperm(users + 4, generator=g)[:users, None].expand(-1, 3).contiguous().int().cuda()  # one block each
    if users > 10:
        table[7] = table[3]  # two users of one block
    for round_ in range(3):
        pos = torch.randint(-1, 3 * bs, (users,), generator=g).cuda()
        for interleaved in (False, True):
            for weights in ((qw, kw), (None, None)):
                got = torch.ops.tt.qk_norm_rope_update_fp8_(q, k, v, angles, pos, *one, table, *weights, b1, 1e-6, interleaved)
                a, turned = torch.ops.tt.qk_norm_rope(q, k, angles, pos, *weights, 1e-6, interleaved)
                torch.ops.tt.paged_update_fp8_cache_(*two, turned[None], v[None], pos, table, b2)
                assert torch.equal(got, a)
                assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((*one, b1), (*two, b2)))


@pytest.mark.parametrize("hkv, d, bs", SHAPES + [(2, 128, 256), (1, 256, 512), (2, 64, 4096), (5, 64, 16), (3, 128, 16), (2, 128, 32), (7, 64, 64),
                                                    (1, 64, 48), (9, 64, 128), (2, 256, 64)])
@pytest.mark.parametrize("users, blocks, short", [(1, 1, 1), (1, 2, 0), (3, 2, 5), (2, 3, -1)])
@pytest.mark.parametrize("bounds", [False, True])
def test_prompts(hkv, d, bs, users, blocks, short, bounds):
    tokens = {1: 1, 0: 2 * bs, 5: bs + 5, -1: 3 * bs - 1}[short]
    nb = users * (blocks + 1) + 2
    cache, b, g = _noise(nb, hkv, bs, d, tokens, bounds)
    table = torch.randperm(nb, generator=g)[: users * (blocks + 1)].view(users, -1).int()
    if users > 2:
        table[1, 0], table[2, 1] = -1, nb  # blocks outside the cache
    rows = torch.randperm(users, generator=g)
    x = [(torch.randn(users, tokens, hkv, d, generator=g) * 2.0 ** torch.randint(-8, 8, (users, 1, hkv, 1), generator=g)).to(torch.bfloat16)
         for _ in range(2)]
    x[0][0, 0, 0, 0], x[0][0, tokens // 2, hkv - 1, 5] = float("nan"), float("inf")
    k, v = (t.transpose(1, 2) for t in x)
    want = R.Cache(*cache, b)
    want.fill(k, v, table, rows.tolist())
    torch.ops.tt.paged_fill_fp8_cache_(*cache, k.cuda(), v.cuda(), table.cuda(), rows.cuda(), b)
    _same(want, cache, b)


def test_a_prompt_without_rows_of_its_own_and_rows_outside_the_table():
    cache, b, g = _noise(6, 2, 32, 64, 1)
    want = R.Cache(*cache, b)
    k = torch.randn(2, 2, 40, 64, generator=g).to(torch.bfloat16)
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32)
    want.fill(k[:1], k[1:], table, [0])
    torch.ops.tt.paged_fill_fp8_cache_(*cache, k[:1].cuda(), k[1:].cuda(), table.cuda(), None, b)
    _same(want, cache, b)
    torch.ops.tt.paged_fill_fp8_cache_(*cache, k.cuda(), k.cuda(), table.cuda(), torch.tensor([-1, 2]).cuda(), b)
    torch.ops.tt.paged_fill_fp8_cache_(*cache, k[:, :, :0].cuda(), k[:, :, :0].cuda(), table.cuda(), torch.tensor([0, 1]).cuda(), b)
    torch.ops.tt.paged_update_fp8_cache_(*cache, k[:1, :0].transpose(1, 2)[:, :0].reshape(1, 0, 2, 64).cuda(),
                                         k[:1, :0].reshape(1, 0, 2, 64).cuda(), torch.empty(0, dtype=torch.int32).cuda(), table.cuda(), b)
    _same(want, cache, b)


def test_a_cache_beyond_four_gibibytes():
    hkv, d, bs = 8, 128, 64
    nb = (1 << 32) // (hkv * d * bs) + 9
    cache = [torch.empty(nb, hkv, bs, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(nb, hkv, device="cuda") for _ in range(2)]
    few = [nb - 1, 3, nb - 2]
    for c in cache:
        c.view(torch.uint8)[few] = 0
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, hkv, 2 * bs + 1, d, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([few], dtype=torch.int32)
    small = [c.view(torch.uint8)[few].view(torch.float8_e4m3fn) for c in cache]
    want = R.Cache(*small, *(s[few] for s in scales))
    order = torch.tensor([[0, 1, 2]])
    want.fill(k, v, order, [0])
    want.update(k[:, :, 5], v[:, :, 5], torch.tensor([2 * bs + 1]), order)
    torch.ops.tt.paged_fill_fp8_cache_(*cache, *scales, k.cuda(), v.cuda(), table.cuda())
    torch.ops.tt.paged_update_fp8_cache_(*cache, *scales, k[:, :, 5].cuda()[None], v[:, :, 5].cuda()[None], torch.tensor([2 * bs + 1]).cuda(), table.cuda())
    got = [c.view(torch.uint8)[few].view(torch.float8_e4m3fn) for c in cache]
    _same(want, (*got, *(s[few] for s in scales)))


def test_refusals():
    cache, b, _ = _noise(4, 2, 32, 64, 1)
    k = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    idx, table = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    ke, ve, ks, vs = cache
    up = torch.ops.tt.paged_update_fp8_cache_
    for args in [
        (ke.view(torch.uint8), ve, ks, vs, k, k, idx, table), (ke, ve[:2], ks, vs, k, k, idx, table), (ke, ve, ks.double(), vs, k, k, idx, table),
        (ke, ve, ks, vs[:2], k, k, idx, table), (ke, ve, ks, vs, k.half(), k, idx, table), (ke, ve, ks, vs, k[:, :2], k, idx, table),
        (ke, ve, ks, vs, k[:, :, :1], k, idx, table), (ke, ve, ks, vs, k, k, idx, table[:2]), (ke, ve, ks, vs, k, k, idx.float(), table),
        (ke, ve, ks, vs, k, k, idx, table, b[:2]), (ke, ve, ks, vs, k, k, idx, table, b.float()), (ke, ve, ks, vs, k, k, idx, table[:, :0]),
        (ke.transpose(2, 3), ve.transpose(2, 3), ks, vs, k, k, idx, table),
    ]:
        with pytest.raises(ValueError):
            up(*args)
    odd = torch.zeros(4, 2, 24, 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        up(odd, odd.clone(), ks, vs, k, k, idx, table)
    fill = torch.ops.tt.paged_fill_fp8_cache_
    p = torch.zeros(2, 2, 65, 64, dtype=torch.bfloat16, device="cuda")
    for args in [(p, p, table, idx[:2]), (p[:, :, :5], p[:, :, :6], table, idx[:2]), (p[:, :, :5], p[:, :, :5], table),
                 (p[:, :, :5], p[:, :, :5], table, idx)]:
        with pytest.raises(ValueError):
            fill(*cache, *args)
    with pytest.raises(NotImplementedError):
        fill(*cache, p[:1, :, :5].clone().requires_grad_(), p[:1, :, :5], table)


def test_one_row_of_the_table_filled_twice_and_one_tensor_for_both_caches():
    hkv, d, bs = 2, 128, 32
    cache, b, g = _noise(20, hkv, bs, d, 3)
    want = R.Cache(*cache, b)
    k, v = (torch.randn(70, hkv, 3 * bs - 5, d, generator=g).to(torch.bfloat16) for _ in range(2))
    table = torch.arange(15, dtype=torch.int32).view(5, 3)
    rows = torch.tensor([2, 4, 2, 9] + [1] * 60 + [4, 0, -1, 2, 1, 9])
    last = [max(i for i, r in enumerate(rows.tolist()) if r == row) for row in range(5) if row in rows.tolist()]
    want.fill(k[last], v[last], table, rows[last])
    torch.ops.tt.paged_fill_fp8_cache_(*cache, k.cuda(), v.cuda(), table.cuda(), rows.cuda(), b)
    assert want.differences(*cache, b) == {}
    ke, ve, ks, vs = cache
    idx = torch.zeros(5, dtype=torch.int32, device="cuda")
    both = torch.zeros(30, hkv, bs, d, dtype=torch.uint8, device="cuda").view(ke.dtype)
    for bad in [(ke, ke, ks, vs), (ke, ve, ks, ks), (both[:20], both[10:], ks, vs)]:
        with pytest.raises(ValueError, match="share"):
            torch.ops.tt.paged_update_fp8_cache_(*bad, k[None, :5, :, 0].cuda(), v[None, :5, :, 0].cuda(), idx, table.cuda())
        with pytest.raises(ValueError, match="share"):
            torch.ops.tt.paged_fill_fp8_cache_(*bad, k[:1].cuda(), v[:1].cuda(), table.cuda())
