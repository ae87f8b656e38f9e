"""The operators around the 8-bit cache together, as a serving program runs them: prompts, chunks and steps through the attention
backend; steps with norm, rotation and write in one launch, sparse steps, captured steps, several streams.  The caches are compared with
their definition (equal), attention with softmax in 64 bits over what the caches stand for (tolerance as in the operators' own tests)."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R
from test_gpu_fp8_chunk import _check as check_chunk
from test_gpu_fp8_decode import _bounds, _check, _check_sparse, _setup

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _layer(nb, hkv, bs, d, bounds=True):
    from tt_xla_amd import TTAttentionBackend as B, fp8_ops

    k, ks = fp8_ops.fp8_empty_cache(nb, hkv, bs, d, "cuda")
    v, vs = fp8_ops.fp8_empty_cache(nb, hkv, bs, d, "cuda")
    b = fp8_ops.fp8_empty_key_bounds(nb, hkv, d, "cuda")
    assert tuple(k.shape) == B.get_kv_cache_storage_shape(nb, bs, hkv, d, "fp8_e4m3")
    assert tuple(ks.shape) == B.get_kv_cache_scale_shape(nb, hkv) and tuple(b.shape) == B.get_kv_cache_bounds_shape(nb, hkv, d)
    return [k, v, ks, vs, b] if bounds else [k, v, ks, vs]


@pytest.mark.parametrize("hq, hkv, d, bs", [(8, 2, 64, 32), (32, 8, 128, 64), (4, 4, 256, 32)])
@pytest.mark.parametrize("sparse", [None, 3])
@pytest.mark.parametrize("aligned", [True, False])
def test_backend_prompt_chunk_and_steps(hq, hkv, d, bs, sparse, aligned):
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    users, first, chunk, steps = 2, 2 * bs, bs, bs + 3
    g = torch.Generator().manual_seed(d)
    width = 6
    kv = _layer(users * width + 1, hkv, bs, d)
    want = R.Cache(*kv)
    table = (torch.randperm(users * width, generator=g) + 1).view(users, width).int()
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8_e4m3", sparse_kept_blocks=sparse)
    assert impl.kv_cache_quantized_dtype == torch.float8_e4m3fn
    batch_idx = torch.arange(users, dtype=torch.int32).cuda()

    def tokens(n):
        return [torch.randn(users, n, h, d, generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv)]

    def forward(q, k, v, meta):
        n = q.shape[0] * q.shape[1] * hq * d
        out = torch.empty(n, dtype=torch.bfloat16, device="cuda") if aligned else torch.empty(n + 1, dtype=torch.bfloat16, device="cuda")[1:]
        impl.forward(None, *(t.flatten(0, 1).flatten(1).cuda() for t in (q, k, v)), kv, meta, output=out.view(-1, hq * d))
        return out.cpu().view(q.shape)

    want.b = torch.zeros(users * width + 1, hkv, 2, d, dtype=torch.float64)
    # a first chunk attends its own keys and values as they are
    q, k, v = tokens(first)
    out = forward(q, k, v, TTMetadata(page_table=table.cuda(), batch_idx=batch_idx, num_users=users))
    want.fill(k.transpose(1, 2), v.transpose(1, 2), table, range(users))
    assert want.differences(*kv) == {}
    allowed = torch.arange(first)[None, :] <= torch.arange(first)[:, None]
    for h in range(0, hq, 3):
        one, size = R.softmax_rows(q[1, :, h], k[1, :, h * hkv // hq].double(), v[1, :, h * hkv // hq].double(), allowed, d**-0.5)
        assert bool(((out[1, :, h].double() - one).abs() <= 2.0**-8 * one.abs() + 0.0085 * size).all())
    # a continuation chunk attends the cache
    q, k, v = tokens(chunk)
    rolled = torch.roll(table, -(first // bs), 1)
    out = forward(q, k, v, TTMetadata(page_table=table.cuda(), fill_page_table=rolled.contiguous().cuda(), batch_idx=batch_idx, num_users=users,
                                      chunk_start_idx=torch.tensor([first], dtype=torch.int32).cuda(), chunk_end=first + chunk))
    want.fill(k.transpose(1, 2), v.transpose(1, 2), rolled, range(users))
    assert want.differences(*kv) == {}
    cache = [t.cpu() for t in kv[:4]]
    check_chunk(out.transpose(1, 2), q.transpose(1, 2), cache, table, first, d**-0.5)
    # steps; a padded row among them
    pad = torch.zeros(1, width, dtype=torch.int32)
    for s in range(steps):
        q, k, v = (torch.cat([t, t[:1]]) for t in tokens(1))
        pos = torch.tensor([first + chunk + s] * users + [-1], dtype=torch.int32)
        tables = torch.cat([table, pad])
        out = forward(q, k, v, TTMetadata(cache_position=pos.cuda(), page_table=tables.cuda(), num_users=users + 1))
        want.update(k[:, 0], v[:, 0], pos, tables)
        if s % 8 == 0 or s == steps - 1:
            assert want.differences(*kv) == {}
            cache = [t.cpu() for t in kv[:4]]
            chosen = None
            if sparse:
                chosen = [[R.choose(q[u, 0, h * hq // hkv : (h + 1) * hq // hkv], kv[4].cpu(), tables[u].tolist(), h, int(pos[u]) // bs + 1, sparse)
                           for h in range(hkv)] for u in range(users)] + [None]
            _check(out[:, 0], q[:, 0], cache, tables, pos, d**-0.5, columns=chosen)


def test_backend_windows_sinks_and_a_shared_cache():
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    hq, hkv, d, bs, users = 8, 2, 64, 32, 3
    cache, table, cur, q, g = _setup(users, hkv, hq // hkv, d, bs, [100, 5, 64], 3)
    kv = [t.cuda() for t in cache]
    sink = torch.randn(hq, generator=g)
    impl = TTAttentionBackendImpl(hq, d, 0.2, hkv, sliding_window=40, sinks=sink.cuda(), kv_cache_dtype="fp8", kv_sharing_target_layer_name="other")
    out = torch.empty(users, hq * d, dtype=torch.bfloat16, device="cuda")
    new = torch.randn(users, hkv * d, generator=g).to(torch.bfloat16).cuda()
    before = [t.clone() for t in kv]
    impl.forward(None, q.flatten(1).cuda(), new, new, kv, TTMetadata(cache_position=cur.cuda(), page_table=table.cuda(), num_users=users), output=out)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, before))
    _check(out.cpu().view(users, hq, d), q, cache, table, cur, 0.2, 40, sink)
    # a prompt over keys and values that another layer has written
    impl = TTAttentionBackendImpl(hq, d, 0.2, hkv, kv_cache_dtype="fp8", kv_sharing_target_layer_name="other")
    q = torch.randn(32, hq * d, generator=g).to(torch.bfloat16)
    out = torch.empty(32, hq * d, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, q.cuda(), new[:1].repeat(32, 1), new[:1].repeat(32, 1), kv,
                 TTMetadata(page_table=table[:1].cuda(), num_users=1, batch_idx=torch.zeros(1, dtype=torch.int32).cuda()), output=out)
    check_chunk(out.cpu().view(1, 32, hq, d).transpose(1, 2), q.view(1, 32, hq, d).transpose(1, 2), cache, table[:1], 0, 0.2)
    for bad in (dict(is_causal=False), dict(attn_mask=torch.zeros(1, device="cuda"))):
        with pytest.raises(NotImplementedError):
            impl.forward(None, q.cuda(), new, new, kv, TTMetadata(page_table=table.cuda(), num_users=1, **bad), output=out)
    with pytest.raises(ValueError):
        impl.forward(None, q.cuda(), new, new, kv[:2], TTMetadata(page_table=table.cuda(), num_users=1), output=out)


def _step(state, sparse):
    """Norm, rotation, write and attention of one step, as a layer runs them."""
    tt = torch.ops.tt
    q = tt.qk_norm_rope_update_fp8_(state["q"], state["k"], state["v"], state["angles"], state["pos"], *state["kv"][:4], state["table"],
                                    state["qw"], state["kw"], state["kv"][4])
    if sparse:
        return tt.paged_fp8_sparse_attention_decode(q[None], *state["kv"], state["table"], state["pos"], 4)[0]
    return tt.paged_fp8_attention_decode(q[None], *state["kv"][:4], state["table"], state["pos"])


def _state(seed, users=9, hq=16, hkv=4, d=128, bs=32):
    from tt_xla_amd.fp8_ops import rope_table

    lengths = [1 + (37 * u * u) % 400 for u in range(users)]
    cache, table, cur, q, g = _setup(users, hkv, hq // hkv, d, bs, lengths, seed)
    kv = [*cache, _bounds(cache)]
    s = {"q": q, "k": torch.randn(users, hkv, d, generator=g).to(torch.bfloat16), "v": torch.randn(users, hkv, d, generator=g).to(torch.bfloat16),
         "qw": 1 + torch.rand(d, generator=g), "kw": 1 + torch.rand(d, generator=g), "angles": rope_table(512, d), "pos": cur, "table": table}
    on = {n: t.cuda() for n, t in s.items()}
    on["kv"] = [t.cuda() for t in kv]
    return on


@pytest.mark.parametrize("sparse", [False, True])
def test_a_step_of_a_layer(sparse):
    s = _state(1)
    want = R.Cache(*s["kv"])
    turned = R.turn(s["k"].cpu(), s["kw"].cpu(), s["angles"].cpu(), s["pos"].cpu(), 1e-6, False)
    got_k = torch.ops.tt.qk_norm_rope(s["q"], s["k"], s["angles"], s["pos"], s["qw"], s["kw"])
    assert float((got_k[1].cpu().double() - turned).abs().max()) <= 2.0**-7 * float(turned.abs().max())
    want.update(got_k[1], s["v"], s["pos"].cpu(), s["table"].cpu())
    out = _step(s, sparse)
    assert want.differences(*s["kv"]) == {}
    cache, q = [t.cpu() for t in s["kv"][:4]], got_k[0].cpu()
    if sparse:
        _, cols = torch.ops.tt.paged_fp8_sparse_attention_decode(got_k[0][None], *s["kv"], s["table"], s["pos"], 4)
        _check_sparse(out[0].cpu(), cols.cpu(), q, cache, s["kv"][4].cpu(), s["table"].cpu(), s["pos"].cpu(), 4, 128**-0.5)
    else:
        _check(out[0].cpu(), q, cache, s["table"].cpu(), s["pos"].cpu(), 128**-0.5)


@pytest.mark.parametrize("sparse", [False, True])
def test_captured_steps(sparse):
    """Two graphs in one process, replayed between eager steps on other tensors; every replay against an eager step on a copy."""
    states = [_state(2), _state(3, users=5, hq=8, hkv=8)]
    graphs, outs = [], []
    for s in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        start = [t.clone() for t in s["kv"]]
        with torch.cuda.stream(side):
            _step(s, sparse)
        torch.cuda.current_stream().wait_stream(side)
        for t, b in zip(s["kv"], start):
            t.view(torch.uint8).copy_(b.view(torch.uint8))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(s, sparse))
        graphs.append(graph)
    g = torch.Generator().manual_seed(7)
    for n in range(6):
        for s, graph, out in zip(states, graphs, outs):
            s["pos"] += 1
            for t in ("q", "k", "v"):
                s[t].copy_(torch.randn(s[t].shape, generator=g).to(torch.bfloat16))
            s["table"][:, :] = torch.where(s["table"] < 0, 0, s["table"])
            copy = dict(s, kv=[t.clone() for t in s["kv"]])
            graph.replay()
            want = _step(copy, sparse)
            if n % 2:
                torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(s["kv"], copy["kv"]))


def test_calls_on_other_streams():
    """Steps of two layers at once on streams of their own, without waits between them."""
    states = [_state(4), _state(5)]
    want = []
    for s in states:
        copy = dict(s, kv=[t.clone() for t in s["kv"]])
        want.append([_step(copy, True).clone() for _ in range(3)] + [_step(copy, False).clone() for _ in range(3)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for n in range(6):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(_step(s, n < 3))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_equal_calls_give_equal_results():
    s = _state(6)
    first = _step(s, False).clone(), _step(s, True).clone()
    for _ in range(5):
        assert torch.equal(_step(s, False), first[0]) and torch.equal(_step(s, True), first[1])


def test_tracing_sees_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    s = _state(8)
    q = s["q"][None]
    with FakeTensorMode() as mode:
        f = {n: mode.from_tensor(t) for n, t in s.items() if n != "kv"}
        kv = [mode.from_tensor(t) for t in s["kv"]]
        fq = mode.from_tensor(q)
        tt = torch.ops.tt
        assert tt.paged_fp8_attention_decode(fq, *kv[:4], f["table"], f["pos"]).shape == q.shape
        out, cols = tt.paged_fp8_sparse_attention_decode(fq, *kv, f["table"], f["pos"], 4)
        assert out.shape == q.shape and cols.shape == (9, 4, 4) and cols.dtype == torch.int32
        assert tt.qk_norm_rope_update_fp8_(f["q"], f["k"], f["v"], f["angles"], f["pos"], *kv[:4], f["table"]).shape == f["q"].shape
        a, b = tt.qk_norm_rope(f["q"], f["k"], f["angles"], f["pos"])
        assert a.shape == f["q"].shape and b.shape == f["k"].shape


@pytest.mark.parametrize("hq, hkv, d, bs, start, s", [(8, 2, 64, 32, 64, 64), (32, 8, 128, 64, 128, 32), (4, 4, 256, 32, 32, 70)])
@pytest.mark.parametrize("known", [True, False])
def test_a_continuation_chunk_of_a_layer_that_shares_a_cache(hq, hkv, d, bs, start, s, known):
    """Its rows attend the whole prefix and the chunk's keys as the layer that owns the cache has written them, and write nothing."""
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    users, width = 2, -(-(start + s) // bs) + 2
    cache, table, _, _, g = _setup(users, hkv, hq // hkv, d, bs, [width * bs] * users, d + s)
    kv = [t.cuda() for t in cache]
    before = [t.clone() for t in kv]
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8", kv_sharing_target_layer_name="other")
    q = torch.randn(users * s, hq * d, generator=g).to(torch.bfloat16)
    new = torch.randn(users * s, hkv * d, generator=g).to(torch.bfloat16).cuda()
    out = torch.empty(users * s, hq * d, dtype=torch.bfloat16, device="cuda")
    meta = TTMetadata(page_table=table.cuda(), num_users=users, batch_idx=torch.arange(users, dtype=torch.int32).cuda(),
                      chunk_start_idx=torch.tensor([start], dtype=torch.int32).cuda(), chunk_end=start + s if known else None)
    impl.forward(None, q.cuda(), new, new, kv, meta, output=out)
    rows = [t.view(users, s, hq, d).transpose(1, 2) for t in (out.cpu(), q)]
    check_chunk(*rows, cache, table, start, d**-0.5)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, before))


def test_windows_of_continuation_chunks():
    """A window that may leave out a key is refused, and nothing is written; one that cannot is none."""
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    hq, hkv, d, bs, start, s = 8, 2, 64, 32, 96, 32
    cache, table, _, _, g = _setup(1, hkv, hq // hkv, d, bs, [6 * bs], 4)
    kv = [t.cuda() for t in cache]
    q = torch.randn(s, hq * d, generator=g).to(torch.bfloat16)
    k, v = (torch.randn(s, hkv * d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    room = table.shape[1] * bs
    for shared in (None, "other"):
        for window, end in ((1, start + s), (start + s - 1, start + s), (start + s, None), (room - 1, None), (start + s, start + s), (room, None),
                            (room, room + 70)):
            impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, sliding_window=window, kv_cache_dtype="fp8", kv_sharing_target_layer_name=shared)
            own = [t.clone() for t in kv]
            out = torch.zeros(s, hq * d, dtype=torch.bfloat16, device="cuda")
            meta = TTMetadata(page_table=table.cuda(), fill_page_table=table[:, start // bs :].contiguous().cuda(), num_users=1,
                              batch_idx=torch.zeros(1, dtype=torch.int32).cuda(), chunk_start_idx=torch.tensor([start], dtype=torch.int32).cuda(),
                              chunk_end=end)
            if window < min(end or room, room):
                with pytest.raises(NotImplementedError, match="sliding window"):
                    impl.forward(None, q.cuda(), k, v, own, meta, output=out)
                assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(own, kv)) and int(out.count_nonzero()) == 0
                continue
            impl.forward(None, q.cuda(), k, v, own, meta, output=out)
            rows = [t.view(1, s, hq, d).transpose(1, 2) for t in (out.cpu(), q)]
            check_chunk(*rows, [t.cpu() for t in own], table, start, d**-0.5)


@pytest.mark.parametrize("wrong", [dict(bounds=False), dict(sliding_window=40), dict(sinks=True)])
def test_a_refused_sparse_step_writes_nothing(wrong):
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    hq, hkv, d, bs = 8, 2, 64, 32
    cache, table, cur, q, g = _setup(2, hkv, hq // hkv, d, bs, [100, 50], 3)
    kv = [t.cuda() for t in cache] + ([_bounds(cache).cuda()] if wrong.pop("bounds", True) else [])
    if wrong.pop("sinks", False):
        wrong["sinks"] = torch.randn(hq, generator=g).cuda()
    before = [t.clone() for t in kv]
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8", sparse_kept_blocks=2, **wrong)
    new = torch.randn(2, hkv * d, generator=g).to(torch.bfloat16).cuda()
    out = torch.zeros(2, hq * d, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(NotImplementedError, match="sparse"):
        impl.forward(None, q.flatten(1).cuda(), new, new, kv, TTMetadata(cache_position=cur.cuda(), page_table=table.cuda(), num_users=2), output=out)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, before)) and int(out.count_nonzero()) == 0


@pytest.mark.parametrize("tensors", [2, 4, 5])
@pytest.mark.parametrize("shared", [None, "other"])
@pytest.mark.parametrize("start", [None, 64])
@pytest.mark.parametrize("kw", [{}, dict(sliding_window=20), dict(sparse_kept_blocks=4)])
def test_prompts_with_caches_that_are_still_empty(tensors, shared, start, kw):
    """What vLLM runs to see how much memory a pass takes: attention of the pass's own keys and values, as with any other type of cache."""
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    hq, hkv, d, bs, users, s = 8, 2, 64, 32, 2, 64
    kv = _layer(0, hkv, bs, d)[:tensors]
    g = torch.Generator().manual_seed(tensors)
    q = torch.randn(users * s, hq * d, generator=g).to(torch.bfloat16)
    k, v = (torch.randn(users * s, hkv * d, generator=g).to(torch.bfloat16) for _ in range(2))
    meta = TTMetadata(page_table=torch.zeros(users, 4, dtype=torch.int32).cuda(), num_users=users, batch_idx=torch.arange(users, dtype=torch.int32).cuda(),
                      chunk_start_idx=None if start is None else torch.tensor([start], dtype=torch.int32).cuda())
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8", kv_sharing_target_layer_name=shared, **kw)
    out = torch.zeros(users * s, hq * d, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, q.cuda(), k.cuda(), v.cuda(), kv, meta, output=out)
    got, q = (t.view(users, s, hq, d) for t in (out.cpu(), q))
    k, v = (t.view(users, s, hkv, d).double() for t in (k, v))
    at = torch.arange(s)
    allowed = (at[None, :] <= at[:, None]) & (at[None, :] > at[:, None] - kw.get("sliding_window", s))
    for u in range(users):
        for h in range(hq):
            one, size = R.softmax_rows(q[u, :, h], k[u, :, h * hkv // hq], v[u, :, h * hkv // hq], allowed, d**-0.5)
            assert bool(((got[u, :, h].double() - one).abs() <= 2.0**-8 * one.abs() + 0.0085 * size).all())


@pytest.mark.parametrize("kind", ["bfloat16", "block-float-8"])
@pytest.mark.parametrize("s", [1, 32])
def test_sparse_passes_over_other_caches_are_refused(kind, s):
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata, custom_ops

    hq, hkv, d, bs, nb = 8, 2, 64, 32, 6
    shape, dtype = ((nb, hkv, bs, d), torch.bfloat16) if kind == "bfloat16" else (custom_ops.bfp8_cache_shape(nb, hkv, bs, d), torch.uint8)
    kv = [torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2)]
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, sparse_kept_blocks=2)
    q, k = (torch.ones(s, h * d, dtype=torch.bfloat16, device="cuda") for h in (hq, hkv))
    out = torch.zeros_like(q)
    meta = TTMetadata(cache_position=torch.zeros(1, dtype=torch.int32).cuda(), page_table=torch.zeros(1, 4, dtype=torch.int32).cuda(), num_users=1,
                      batch_idx=torch.zeros(1, dtype=torch.int32).cuda())
    with pytest.raises(NotImplementedError, match="sparse"):
        impl.forward(None, q, k, k, kv, meta, output=out)
    assert not any(int(t.count_nonzero()) for t in (*kv, out))


def _odd(t):
    """The same values in a contiguous tensor whose address is no multiple of 16."""
    x = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
    x.copy_(t)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


def test_operands_at_odd_addresses():
    """Contiguous tensors that vector loads cannot take: the results of aligned ones, in place and in the caches too."""
    tt, s = torch.ops.tt, _state(9)
    users = s["q"].shape[0]
    g = torch.Generator().manual_seed(12)
    rope = [s[n] for n in ("q", "k", "angles", "pos", "qw", "kw")]
    odd = [_odd(t) if t.is_floating_point() else t for t in rope]
    want = tt.qk_norm_rope(*rope)
    for i in range(len(rope)):
        got = tt.qk_norm_rope(*rope[:i], odd[i], *rope[i + 1 :])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q, k = _odd(s["q"]), _odd(s["k"])
    tt.qk_norm_rope_(q, k, *rope[2:])
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])

    def same(call, *args):
        """call(caches, *args) gives the same results and caches whichever operand lies at an odd address."""
        def once(*a):
            kv = [t.clone() for t in s["kv"]]
            out = call(kv, *a)
            return [t for t in (out if isinstance(out, (list, tuple)) else [out]) if t is not None] + kv

        want = once(*args)
        for i in range(len(args)):
            got = once(*args[:i], _odd(args[i]), *args[i + 1 :])
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want)), i

    table, pos = s["table"], s["pos"]
    same(lambda kv, q, k, v: tt.qk_norm_rope_update_fp8_(q, k, v, s["angles"], pos, *kv[:4], table, s["qw"], s["kw"], kv[4]), s["q"], s["k"], s["v"])
    same(lambda kv, k, v: tt.paged_update_fp8_cache_(*kv[:4], k, v, pos, table, kv[4]), s["k"][None], s["v"][None])
    prompts = [torch.randn(2, 4, 45, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    same(lambda kv, k, v: tt.paged_fill_fp8_cache_(*kv[:4], k, v, table[:2, :2].contiguous(), torch.tensor([1, 0]).cuda(), kv[4]), *prompts)
    same(lambda kv, q: tt.paged_fp8_attention_decode(q, *kv[:4], table, pos), s["q"][None])
    same(lambda kv, q: tt.paged_fp8_sparse_attention_decode(q, *kv, table, pos, 3), s["q"][None])
    rows = torch.randn(users, 16, 40, 128, generator=g).to(torch.bfloat16).cuda()
    same(lambda kv, q: tt.chunked_fp8_attention(q, *kv[:4], table, torch.tensor([20]).cuda()), rows)
    sink = torch.randn(16, generator=g).cuda()
    same(lambda kv, x: tt.paged_fp8_attention_decode(s["q"][None], *kv[:4], table, pos, x), sink)


@pytest.mark.parametrize("form", ["few", "copies"])
def test_outputs_in_the_memory_of_the_query(form, monkeypatch):
    """The query itself and views beside it are written; what would overwrite rows that are still to be read is refused."""
    monkeypatch.setenv("TTPA_CHUNK_FORM", form)
    tt, s = torch.ops.tt, _state(13)
    users, hq, d = s["q"].shape
    g = torch.Generator().manual_seed(14)
    rows, start = torch.randn(users, hq, 40, d, generator=g).to(torch.bfloat16).cuda(), torch.tensor([20]).cuda()
    calls = [(s["q"][None], lambda q, out: tt.paged_fp8_attention_decode_out(q, *s["kv"][:4], s["table"], s["pos"], out)),
             (s["q"][None], lambda q, out: tt.paged_fp8_sparse_attention_decode_out(q, *s["kv"], s["table"], s["pos"], out, 3)),
             (rows, lambda q, out: tt.chunked_fp8_attention_out(q, *s["kv"][:4], s["table"], start, out))]
    for q, call in calls:
        want = torch.empty_like(q)
        call(q, want)
        own = q.clone()
        call(own, own)
        assert torch.equal(own.view(torch.int16), want.view(torch.int16))

        def views():
            """(query, out, whether that can be served): two views of one memory."""
            for dim in range(1, q.dim()):
                size = q.shape[dim]
                both = torch.cat([q, q], dim).contiguous()
                yield both.narrow(dim, 0, size), both.narrow(dim, size, size), True
                if size > 1:
                    yield both.narrow(dim, size, size), both.narrow(dim, 1, size), False
                    yield both.narrow(dim, 0, size), both.narrow(dim, 1, size), False
            two = torch.stack([q, q], -2)
            yield two[..., 0, :], two[..., 1, :], True
            flat = torch.cat([q.flatten(), q.flatten()])
            yield flat[: q.numel()].view(q.shape), flat[q.numel() :].view(q.shape), True
            yield flat[: q.numel()].view(q.shape), flat[d : q.numel() + d].view(q.shape), False
            yield flat[: q.numel()].view(q.shape), flat[8 : q.numel() + 8].view(q.shape), False
            swapped = (q.shape[0], q.shape[2], q.shape[1], d)
            yield flat[: q.numel()].view(q.shape), flat[: q.numel()].view(swapped).transpose(1, 2), False

        for query, out, served in views():
            if served:
                query.copy_(q)
                call(query, out)
                assert torch.equal(out.contiguous().view(torch.int16), want.contiguous().view(torch.int16)) and torch.equal(query, q)
            else:
                with pytest.raises(ValueError, match="overlap"):
                    call(query, out)


def test_block_ids_and_starts_beyond_32_bits():
    """Numbers that lose their upper half would name a block of the cache, or a start in it: they are outside, like other ids that are too large."""
    tt, hq, hkv, d, bs = torch.ops.tt, 8, 2, 64, 32
    cache, table, cur, q, g = _setup(2, hkv, hq // hkv, d, bs, [100, 70], 3)
    bounds = _bounds(cache)
    kv, b = [t.cuda() for t in cache], bounds.cuda()
    before = [t.clone() for t in (*kv, b)]
    for far in (1 << 32, -(1 << 32)):
        ids = table.long() + far
        x = torch.randn(2, hkv, d, generator=g).to(torch.bfloat16).cuda()
        tt.paged_update_fp8_cache_(*kv, x[None], x[None], cur.cuda(), ids.cuda(), b)
        prompt = torch.randn(2, hkv, 40, d, generator=g).to(torch.bfloat16).cuda()
        tt.paged_fill_fp8_cache_(*kv, prompt, prompt, ids.cuda(), torch.arange(2).cuda(), b)
        assert all(torch.equal(a.view(torch.uint8), c.view(torch.uint8)) for a, c in zip((*kv, b), before))
        zeros = torch.zeros_like(table)  # what is outside the cache reads block 0
        out = tt.paged_fp8_attention_decode(q.cuda()[None], *kv, ids.cuda(), cur.cuda())[0].cpu()
        _check(out, q, cache, zeros, cur, d**-0.5)
        out, cols = tt.paged_fp8_sparse_attention_decode(q.cuda()[None], *kv, b, ids.cuda(), cur.cuda(), 3)
        _check_sparse(out[0].cpu(), cols.cpu(), q, cache, bounds, zeros, cur, 3, d**-0.5)
    rows = torch.randn(2, hq, 20, d, generator=g).to(torch.bfloat16)
    ids = table.clamp(min=0)
    room = ids.shape[1] * bs
    out = tt.chunked_fp8_attention(rows.cuda(), *kv, ids.cuda(), torch.tensor([1 << 32]).cuda()).cpu()
    check_chunk(out, rows, cache, ids, room, d**-0.5)
    assert torch.isnan(tt.chunked_fp8_attention(rows.cuda(), *kv, ids.cuda(), torch.tensor([-(1 << 32)]).cuda())).all()


@pytest.mark.parametrize("sparse", [None, 3])
def test_captured_passes_of_the_backend(sparse):
    """A prompt, a continuation chunk of an owning and of a sharing layer and a step in one graph, replayed with other tokens, places and starts;
    every replay against the eager passes on a copy."""
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    hq, hkv, d, bs, users, s = 8, 2, 128, 32, 2, 64
    g = torch.Generator().manual_seed(21)
    cache, table, _, _, _ = _setup(users, hkv, hq // hkv, d, bs, [10 * bs] * users, 5)
    kv, table = [t.cuda() for t in (*cache, _bounds(cache))], table.cuda()
    fill, rows, start = table[:, :2].contiguous(), torch.arange(users, dtype=torch.int32).cuda(), torch.tensor([4 * bs], dtype=torch.int32).cuda()
    place, pos = table[:, 4:6].contiguous(), torch.tensor([6 * bs, 7 * bs + 5], dtype=torch.int32).cuda()
    own = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8", sparse_kept_blocks=sparse)
    sharing = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8", kv_sharing_target_layer_name="other")
    tokens = {n: [torch.randn(users * n, h * d, generator=g).to(torch.bfloat16).cuda() for h in (hq, hkv, hkv)] for n in (1, s)}

    def passes(kv):
        out = [torch.zeros(users * n, hq * d, dtype=torch.bfloat16, device="cuda") for n in (s, s, s, 1)]
        one = dict(page_table=table, batch_idx=rows, num_users=users)
        own.forward(None, *tokens[s], kv, TTMetadata(fill_page_table=fill, **one), output=out[0])
        own.forward(None, *tokens[s], kv, TTMetadata(fill_page_table=place, chunk_start_idx=start, **one), output=out[1])
        sharing.forward(None, *tokens[s], kv, TTMetadata(fill_page_table=place, chunk_start_idx=start, **one), output=out[2])
        own.forward(None, *tokens[1], kv, TTMetadata(page_table=table, cache_position=pos, num_users=users), output=out[3])
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes([t.clone() for t in kv])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = passes(kv)
    for n, at in enumerate((4, 2, 6, 0, 8)):
        start.fill_(at * bs)
        place.copy_(table[:, at : at + 2])
        pos.copy_(torch.tensor([n * 40, -1 if n == 2 else 200 + n]))
        for ts in tokens.values():
            for t in ts:
                t.copy_(torch.randn(t.shape, generator=g).to(torch.bfloat16))
        copy = [t.clone() for t in kv]
        graph.replay()
        want = passes(copy)
        if n % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want)), n
        assert torch.equal(want[1], want[2])  # (the sharing layer sees what the owner has written)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, copy))
