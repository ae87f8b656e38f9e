"""Norm and rotation by positions on several axes (``tt::qk_norm_rope_axes``, ``tt::qk_norm_rope_axes_``) against the same in 64 bits.

Tolerance: as for one axis, whose arithmetic it is (a rounding to bfloat16, 2^-8 of the result, and less than 32 half units of the
two products of float32 values before it, 2^-19 of twice the row's largest result)."""

import pytest
import torch

import __graft_entry__ as entry
import media_reference as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _table(positions, rotary, dtype=torch.float32):
    from tt_xla_amd.fp8_ops import rope_table

    return rope_table(positions, rotary, 10000.0, "cpu", dtype)


def _check(got, x, weight, table, pos, pairs, eps, interleaved):
    want = M.turn_axes(x, weight, table, pos, pairs, eps, interleaved)
    size = 2 * want.abs().amax(-1, keepdim=True)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= 2.0**-8 * want.abs() + 2.0**-19 * size + 2.0**-126).all()), float((err - 2.0**-8 * want.abs()).max())


def _pair_axes(kind, pairs, axes):
    from tt_xla_amd.media_ops import rope_pair_axes

    if kind == "sections":  # borders at odd pairs
        first = pairs // axes // 2 * 2 + 1 if axes > 1 else pairs
        rest = [(pairs - first) // (axes - 1)] * (axes - 1) if axes > 1 else []
        if rest:
            rest[-1] += pairs - first - sum(rest)
        return rope_pair_axes([first, *rest])
    if kind == "alternating":
        each = pairs // axes
        return rope_pair_axes([pairs - each * (axes - 1)] + [each] * (axes - 1), alternating=True)
    return torch.randint(-1, axes + 1, (pairs,), generator=torch.Generator().manual_seed(pairs)).int()  # some axes do not exist


@pytest.mark.parametrize("tokens", [1, 3, 37, 700])
@pytest.mark.parametrize("hq, hk, d, rotary", [(8, 2, 64, 64), (32, 8, 128, 128), (5, 1, 128, 64), (16, 8, 256, 256), (3, 3, 256, 96), (7, 2, 64, 16)])
@pytest.mark.parametrize("kind, axes", [("sections", 3), ("alternating", 3), ("sections", 2), ("any", 4), ("sections", 1)])
def test_rows(tokens, hq, hk, d, rotary, kind, axes):
    g = torch.Generator().manual_seed(tokens * 1000 + hq)
    qkv = torch.randn(tokens, (hq + 2 * hk) * d, generator=g).to(torch.bfloat16)
    table, pairs = _table(300, rotary), _pair_axes(kind, rotary // 2, axes)
    pos = torch.randint(-2, 304, (axes, tokens), generator=g, dtype=torch.int32)
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g)).to(torch.bfloat16), 1 + 0.3 * torch.randn(d, generator=g)
    dev = qkv.cuda()
    split = lambda x: [t.unflatten(1, (-1, d)) for t in x.split([hq * d, hk * d, hk * d], 1)]  # noqa: E731
    q, k, _ = split(dev)
    for interleaved in (False, True):
        for weights in ((qw, kw), (None, None)):
            on = [None if w is None else w.cuda() for w in weights]
            a, b = torch.ops.tt.qk_norm_rope_axes(q, k, table.cuda(), pos.cuda(), pairs.cuda(), *on, 1e-5, interleaved)
            _check(a, q.cpu(), weights[0], table, pos, pairs, 1e-5, interleaved)
            _check(b, k.cpu(), weights[1], table, pos, pairs, 1e-5, interleaved)
            own = dev.clone()
            q2, k2, v2 = split(own)
            torch.ops.tt.qk_norm_rope_axes_(q2, k2, table.cuda(), pos.cuda(), pairs.cuda(), *on, 1e-5, interleaved)
            assert torch.equal(q2, a) and torch.equal(k2, b) and torch.equal(v2, split(dev)[2])


@pytest.mark.parametrize("hq, hk, d, rotary, tokens", [(8, 2, 64, 32, 8195), (8, 1, 128, 128, 4100), (2, 2, 256, 256, 8192), (40, 8, 128, 128, 1367), (48, 8, 128, 128, 1171),
                                                       (32, 8, 128, 64, 2053), (16, 8, 256, 256, 1366)])
@pytest.mark.parametrize("kind", ["sections", "alternating"])
def test_many_tokens(hq, hk, d, rotary, tokens, kind):
    """Every form of the kernel: rows of neighbouring tokens in a wavefront, three to five groups of heads in one."""
    g = torch.Generator().manual_seed(tokens + hq)
    both = torch.randn(tokens, hq + hk + 1, d, generator=g).to(torch.bfloat16)
    q, k = both[:, :hq], both[:, hq : hq + hk]
    table, pairs = _table(300, rotary), _pair_axes(kind, rotary // 2, 3)
    pos = torch.randint(-2, 305, (3, tokens), generator=g)
    qw = 1 + 0.2 * torch.randn(d, generator=g)
    on = both.cuda()
    got = torch.ops.tt.qk_norm_rope_axes(on[:, :hq], on[:, hq : hq + hk], table.cuda(), pos.cuda(), pairs.cuda(), qw.cuda(), None)
    _check(got[0], q, qw, table, pos, pairs, 1e-6, False)
    _check(got[1], k, None, table, pos, pairs, 1e-6, False)


@pytest.mark.parametrize("kind", ["sections", "alternating"])
def test_equal_positions_on_all_axes_are_one_position(kind):
    """Text: the results of the operator with one axis, bit for bit."""
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(50, 8, 128, generator=g).to(torch.bfloat16).cuda(), torch.randn(50, 2, 128, generator=g).to(torch.bfloat16).cuda()
    pos, w = torch.randint(0, 100, (50,), generator=g).cuda(), torch.rand(128, generator=g).cuda()
    table, pairs = _table(100, 128).cuda(), _pair_axes(kind, 64, 3).cuda()
    want = torch.ops.tt.qk_norm_rope(q, k, table, pos, w, w)
    got = torch.ops.tt.qk_norm_rope_axes(q, k, table, pos.expand(3, -1), pairs, w, w)  # (one row of positions for all axes)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_table_in_bfloat16_far_positions_and_other_integers():
    g = torch.Generator().manual_seed(4)
    q, k = torch.randn(5, 4, 128, generator=g).to(torch.bfloat16), torch.randn(5, 2, 128, generator=g).to(torch.bfloat16)
    pos = torch.tensor([[0, 69999, -1, 1 << 40, 3], [5, 1, 70000, 2, 3], [9, 9, 9, 9, 3]])
    pairs = _pair_axes("sections", 64, 3)
    for dtype in (torch.float32, torch.bfloat16):
        table = _table(70000, 128, dtype)
        a, b = torch.ops.tt.qk_norm_rope_axes(q.cuda(), k.cuda(), table.cuda(), pos.cuda(), pairs.cuda().long())
        _check(a, q, None, table, pos, pairs, 1e-6, False)
        _check(b, k, None, table, pos, pairs, 1e-6, False)
    short = pos.clamp(-1, 100).to(torch.int16)
    a, _ = torch.ops.tt.qk_norm_rope_axes(q.cuda(), k.cuda(), table.cuda(), short.cuda(), pairs.cuda().to(torch.int8))
    _check(a, q, None, table, short.long(), pairs, 1e-6, False)


def test_strides_and_bases_that_vector_loads_cannot_take():
    g = torch.Generator().manual_seed(5)
    base = torch.randn(3 * (5 * 64 + 3) + 1, generator=g).to(torch.bfloat16).cuda()
    q = base[1:].as_strided((3, 3, 64), (5 * 64 + 3, 64, 1), 1)
    k = base[1:].as_strided((3, 2, 64), (5 * 64 + 3, 64, 1), 1 + 3 * 64)
    table = _table(8, 64).cuda()
    pos = torch.randint(0, 8, (3, 2, 3), generator=g).cuda()[:, 0].transpose(0, 1)  # [axes, tokens] by odd strides
    pairs = torch.cat([torch.zeros(1), _pair_axes("any", 32, 3)]).int().cuda()[1:]    # an odd base
    want = torch.ops.tt.qk_norm_rope_axes(q.contiguous(), k.contiguous(), table, pos.contiguous(), pairs.clone())
    got = torch.ops.tt.qk_norm_rope_axes(q, k, table, pos, pairs)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    torch.ops.tt.qk_norm_rope_axes_(q, k, table, pos, pairs)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_no_tokens():
    q, k = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    a, b = torch.ops.tt.qk_norm_rope_axes(q, k, _table(4, 64).cuda(), torch.empty(3, 0, dtype=torch.int32, device="cuda"), _pair_axes("any", 32, 3).cuda())
    assert a.shape == q.shape and b.shape == k.shape


def test_refusals():
    z = dict(device="cuda")
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16, **z), torch.zeros(2, 2, 64, dtype=torch.bfloat16, **z)
    table, pos, pairs = _table(4, 64).cuda(), torch.zeros(3, 2, dtype=torch.int32, **z), torch.zeros(32, dtype=torch.int32, **z)
    for op in (torch.ops.tt.qk_norm_rope_axes, torch.ops.tt.qk_norm_rope_axes_):
        for args in [(q.float(), k, table, pos, pairs), (q[0], k, table, pos, pairs), (q, k, table.half(), pos, pairs), (q, k, table, pos[0], pairs),
                     (q, k, table, pos[:, :1], pairs), (q, k, table, pos.float(), pairs), (q, k, table, pos, pairs[:31]), (q, k, table, pos, pairs.float()),
                     (q, k, table, pos, pairs[None]), (q, k, table, torch.zeros(5, 2, dtype=torch.int32, **z), pairs), (q, k, table, pos[:0], pairs)]:
            with pytest.raises(ValueError):
                op(*args)
        with pytest.raises(NotImplementedError):
            op(q, k, table, pos, pairs.cpu())
        with pytest.raises(NotImplementedError):
            op(q.clone().requires_grad_(), k, table, pos, pairs)
    with pytest.raises(ValueError, match="overlap"):
        torch.ops.tt.qk_norm_rope_axes_(q, q, table, pos, pairs)


def test_captured_in_place():
    """Replayed at other positions, every replay against the eager call."""
    g = torch.Generator().manual_seed(8)
    table, pairs = _table(200, 128).cuda(), _pair_axes("sections", 64, 3).cuda()
    x = torch.randn(6, 12, 128, generator=g).to(torch.bfloat16).cuda()
    pos = torch.randint(0, 200, (3, 6), generator=g).cuda()
    run = lambda t: torch.ops.tt.qk_norm_rope_axes_(t[:, :8], t[:, 8:10], table, pos, pairs)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(x)
    for n in range(4):
        x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
        pos.copy_(torch.randint(0, 200, (3, 6), generator=g))
        want = x.clone()
        graph.replay()
        run(want)
        assert torch.equal(x, want)
