"""Norms of queries and keys with the position rotation (``tt::qk_norm_rope``, ``tt::qk_norm_rope_``) against the same in
64 bits.

Tolerance: the result is rounded to bfloat16 once, 2^-8 of it; before that a feature is a sum of two products of float32
values, each of which carries the rounding of x * (inv * weight) (two products), of inv (a division, a root and a mean over up to
256 squares in a tree of at most 16 additions in a row) and of the cosine: less than 32 half units, 32 * 2^-24 of the two products' size.  The row's
largest result bounds neither, so the bound is 2^-19 of |y_i| + |y_j| <= 2 max |y| of the normed row, and of the result."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _table(positions, rotary, dtype=torch.float32):
    from tt_xla_amd.fp8_ops import rope_table

    return rope_table(positions, rotary, 10000.0, "cpu", dtype)


def _inputs(tokens, hq, hk, d, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, (hq + 2 * hk) * d, generator=g) * gain).to(torch.bfloat16)
    return qkv, g


def _check(got, x, weight, table, pos, eps, interleaved):
    want = R.turn(x, weight, table, pos, eps, interleaved)
    size = 2 * want.abs().amax(-1, keepdim=True)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= 2.0**-8 * want.abs() + 2.0**-19 * size + 2.0**-126).all()), float((err - 2.0**-8 * want.abs()).max())


@pytest.mark.parametrize("tokens", [1, 2, 37, 700])
@pytest.mark.parametrize("hq, hk, d, rotary", [(8, 2, 64, 64), (32, 8, 128, 128), (5, 1, 128, 64), (16, 8, 256, 256), (3, 3, 256, 96), (7, 2, 64, 16)])
def test_rows(tokens, hq, hk, d, rotary):
    qkv, g = _inputs(tokens, hq, hk, d, tokens * 1000 + hq)
    table = _table(300, rotary)
    pos = torch.randint(0, 300, (tokens,), generator=g, dtype=torch.int32)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g)).to(torch.bfloat16), (1 + 0.3 * torch.randn(d, generator=g)).to(torch.bfloat16)
    dev = qkv.cuda()
    q, k, _ = dev.split([hq * d, hk * d, hk * d], 1)  # views of a projection's output
    q, k = q.unflatten(1, (hq, d)), k.unflatten(1, (hk, d))
    for interleaved in (False, True):
        for weights in ((qw, kw), (None, None), (qw.float(), None)):
            on = [None if w is None else w.cuda() for w in weights]
            a, b = torch.ops.tt.qk_norm_rope(q, k, table.cuda(), pos.cuda(), *on, 1e-5, interleaved)
            _check(a, q.cpu(), weights[0], table, pos, 1e-5, interleaved)
            _check(b, k.cpu(), weights[1], table, pos, 1e-5, interleaved)
            # in place on the views: the same bits, and the values between them untouched
            own = dev.clone()
            q2, k2, v2 = own.split([hq * d, hk * d, hk * d], 1)
            torch.ops.tt.qk_norm_rope_(q2.unflatten(1, (hq, d)), k2.unflatten(1, (hk, d)), table.cuda(), pos.cuda(), *on, 1e-5, interleaved)
            assert torch.equal(q2.unflatten(1, (hq, d)), a) and torch.equal(k2.unflatten(1, (hk, d)), b)
            assert torch.equal(v2, dev[:, (hq + hk) * d :])


@pytest.mark.parametrize("hq, hk, d, rotary, tokens", [(8, 2, 64, 32, 8195), (1, 1, 64, 64, 8200), (8, 1, 128, 128, 4100), (5, 1, 128, 64, 8193), (2, 2, 256, 256, 8192),
                                                       (3, 2, 256, 96, 4111), (14, 3, 128, 128, 2731), (30, 3, 128, 128, 1700), (63, 2, 64, 64, 1650), (25, 3, 128, 96, 2100)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens_of_few_heads(hq, hk, d, rotary, tokens, interleaved):
    """Rows of neighbouring tokens in one wavefront, views of a projection, positions in no order and outside the table."""
    g = torch.Generator().manual_seed(tokens + hq)
    both = torch.randn(tokens, hq + hk + 1, d, generator=g).to(torch.bfloat16)
    q, k = both[:, :hq], both[:, hq : hq + hk]
    table = _table(300, rotary)
    pos = torch.randint(-2, 305, (tokens,), generator=g)
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    on = both.cuda()
    got = torch.ops.tt.qk_norm_rope(on[:, :hq], on[:, hq : hq + hk], table.cuda(), pos.cuda(), qw.cuda(), None, 1e-6, interleaved)
    _check(got[0].cpu(), q, qw, table, pos, 1e-6, interleaved)
    _check(got[1].cpu(), k, None, table, pos, 1e-6, interleaved)
    torch.ops.tt.qk_norm_rope_(on[:, :hq], on[:, hq : hq + hk], table.cuda(), pos.cuda(), qw.cuda(), None, 1e-6, interleaved)
    assert torch.equal(on[:, :hq], got[0]) and torch.equal(on[:, hq : hq + hk], got[1]) and torch.equal(on[:, hq + hk :].cpu(), both[:, hq + hk :])


def test_table_in_bfloat16_long_positions_and_positions_outside():
    tokens, hq, hk, d = 6, 4, 2, 128
    qkv, _ = _inputs(tokens, hq, hk, d, 3)
    q, k = qkv[:, : hq * d].view(tokens, hq, d), qkv[:, hq * d : (hq + hk) * d].reshape(tokens, hk, d)
    for dtype in (torch.float32, torch.bfloat16):
        table = _table(70000, 128, dtype)
        pos = torch.tensor([-1, 0, 1, 69999, 70000, 1 << 40])
        a, b = torch.ops.tt.qk_norm_rope(q.cuda(), k.cuda(), table.cuda(), pos.cuda())
        _check(a, q, None, table, pos, 1e-6, False)
        _check(b, k, None, table, pos, 1e-6, False)
        assert torch.equal(a[0].cpu(), q[0]) and torch.equal(a[4].cpu(), q[4])  # no norm, not turned: a copy


@pytest.mark.parametrize("gain", [0.0, 1e-18, 1e18])
def test_rows_of_zeros_and_of_extreme_size(gain):
    """Squares of 10^18 add up to 10^38 below the largest float; eps keeps rows of zeros finite."""
    qkv, g = _inputs(9, 4, 2, 64, 11, gain)
    q, k = qkv[:, :256].view(9, 4, 64), qkv[:, 256:384].reshape(9, 2, 64)
    w = torch.ones(64, dtype=torch.bfloat16)
    table, pos = _table(16, 64), torch.arange(9)
    a, b = torch.ops.tt.qk_norm_rope(q.cuda(), k.cuda(), table.cuda(), pos.cuda(), w.cuda(), w.cuda(), 1e-30)
    _check(a, q, w, table, pos, 1e-30, False)
    _check(b, k, w, table, pos, 1e-30, False)


def test_rows_that_vector_loads_cannot_take():
    """Odd strides and bases: copies inside the call, the same result in place."""
    g = torch.Generator().manual_seed(5)
    base = torch.randn(3 * (5 * 64 + 3) + 1, generator=g).to(torch.bfloat16).cuda()
    q = base[1:].as_strided((3, 3, 64), (5 * 64 + 3, 64, 1), 1)
    k = base[1:].as_strided((3, 2, 64), (5 * 64 + 3, 64, 1), 1 + 3 * 64)
    table, pos = _table(8, 64), torch.tensor([7, 0, 3])
    want = torch.ops.tt.qk_norm_rope(q.contiguous(), k.contiguous(), table.cuda(), pos.cuda())
    got = torch.ops.tt.qk_norm_rope(q, k, table.cuda(), pos.cuda())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    torch.ops.tt.qk_norm_rope_(q, k, table.cuda(), pos.cuda())
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_no_tokens():
    q, k = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    a, b = torch.ops.tt.qk_norm_rope(q, k, _table(4, 64).cuda(), torch.empty(0, dtype=torch.int32, device="cuda"))
    assert a.shape == q.shape and b.shape == k.shape


def test_refusals():
    z = dict(device="cuda")
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16, **z), torch.zeros(2, 2, 64, dtype=torch.bfloat16, **z)
    table, pos = _table(4, 64).cuda(), torch.zeros(2, dtype=torch.int32, **z)
    op = torch.ops.tt.qk_norm_rope
    bad = [
        (q.float(), k, table, pos), (q, k.half(), table, pos), (q[0], k, table, pos), (q, k[:1], table, pos),
        (q, k, table.half(), pos), (q, k, table[0], pos), (q, k, table[:, :24], pos), (q, k, torch.zeros(4, 80, **z), pos),
        (q, k, table, pos[:1]), (q, k, table, pos.float()), (q, k, table, pos, torch.ones(32, **z)),
        (q, k, table, pos, torch.ones(64, dtype=torch.float64, **z)),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(RuntimeError):  # a head size without a kernel
        op(torch.zeros(2, 4, 96, dtype=torch.bfloat16, **z), torch.zeros(2, 2, 96, dtype=torch.bfloat16, **z), table, pos)
    with pytest.raises(RuntimeError):
        op(q, k, table, pos, None, None, -1.0)
    with pytest.raises(NotImplementedError):
        op(q, k, table.cpu(), pos)
    with pytest.raises(NotImplementedError):
        op(q.clone().requires_grad_(), k, table, pos)
    with torch.no_grad():
        op(q.clone().requires_grad_(), k, table, pos)


def test_operands_that_overlap_are_not_turned_in_place():
    x = torch.zeros(3, 6, 64, dtype=torch.bfloat16, device="cuda")
    table, pos = _table(4, 64).cuda(), torch.zeros(3, dtype=torch.int32, device="cuda")
    op = torch.ops.tt.qk_norm_rope_
    for q, k in [(x[:1].expand(3, -1, -1), x[:, :2].clone()), (x[:, :2].clone(), x[:, :1].expand(-1, 4, -1)), (x, x), (x[:, :4], x[:, :2]),
                 (x[:2], x[1:]), (x[:, :4], x[:, 3:]), (x[:, 2:4], x[:, 1:]), (x[:, ::2], x[:, 1:3]),
                 (x.as_strided((3, 3, 64), (128, 64, 1)), x[:, :2].clone()), (x.as_strided((3, 4, 64), (384, 32, 1)), x[:, :2].clone()),
                 (x.as_strided((3, 4, 64), (64, 64, 1)), x[:, :2].clone()), (x[:, :2].clone(), x.as_strided((3, 2, 64), (8, 128, 1)))]:
        with pytest.raises(ValueError):
            op(q, k, table, pos[: q.shape[0]])


def test_views_of_one_projection_are_turned_in_place():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 6, 64, generator=g).to(torch.bfloat16).cuda()
    table, pos = _table(4, 64).cuda(), torch.tensor([0, 3, 1], dtype=torch.int32, device="cuda")
    op = torch.ops.tt.qk_norm_rope_
    for q, k in [(slice(0, 4), slice(4, 6)), (slice(4, 6), slice(0, 4)), (slice(0, 6, 2), slice(1, 6, 2)), (slice(0, 3), slice(5, 6))]:
        want = torch.ops.tt.qk_norm_rope(x[:, q].contiguous(), x[:, k].contiguous(), table, pos)
        y = x.clone()
        op(y[:, q], y[:, k], table, pos)
        assert torch.equal(y[:, q], want[0]) and torch.equal(y[:, k], want[1])
    y = x.clone()  # (tokens behind tokens)
    want = torch.ops.tt.qk_norm_rope(x[:1], x[1:2], table, pos[:1])
    op(y[:1], y[1:2], table, pos[:1])
    assert torch.equal(y[:1], want[0]) and torch.equal(y[1:2], want[1])


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    table, pos = _table(4, 64).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
        torch.ops.tt.qk_norm_rope(fwd.make_dual(q, torch.ones_like(q)), q, table, pos)


@pytest.mark.parametrize("hq, hk, d, rotary, tokens", [(40, 8, 128, 128, 1367), (64, 8, 128, 64, 911), (32, 32, 128, 128, 1025), (16, 8, 256, 256, 1366), (48, 8, 128, 128, 1171),
                                                       (129, 8, 128, 96, 483), (90, 7, 64, 64, 1173), (21, 3, 256, 32, 1366), (64, 64, 64, 64, 1030)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens_of_many_heads(hq, hk, d, rotary, tokens, interleaved):
    """Several wavefronts per token with several groups of heads in each, the last of them full or not; also in place."""
    g = torch.Generator().manual_seed(tokens + hq)
    both = torch.randn(tokens, hq + hk + 1, d, generator=g).to(torch.bfloat16)
    q, k = both[:, :hq], both[:, hq : hq + hk]
    table = _table(300, rotary)
    pos = torch.randint(-2, 305, (tokens,), generator=g, dtype=torch.int32)
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    on = both.cuda()
    for weights in ((None, kw), (qw, kw.to(torch.bfloat16))):
        w = [None if t is None else t.cuda() for t in weights]
        args = (table.cuda(), pos.cuda(), *w, 1e-6, interleaved)
        got = torch.ops.tt.qk_norm_rope(on[:, :hq], on[:, hq : hq + hk], *args)
        _check(got[0].cpu(), q, weights[0], table, pos, 1e-6, interleaved)
        _check(got[1].cpu(), k, weights[1], table, pos, 1e-6, interleaved)
        own = on.clone()
        torch.ops.tt.qk_norm_rope_(own[:, :hq], own[:, hq : hq + hk], *args)
        assert torch.equal(own[:, :hq], got[0]) and torch.equal(own[:, hq : hq + hk], got[1]) and torch.equal(own[:, hq + hk :].cpu(), both[:, hq + hk :])
