"""Attention to an encoder's states in a paged 8-bit cache (``tt::paged_fp8_cross_attention``) against softmax in 64 bits over the values that the elements stand for.

An element times its block's scale is a bfloat16 value, so the tolerance is that of ``test_gpu_cross_attention.py``: 2^-8 |out| + (2 * 2^-8 * 1.005 + 6e-4) sum p |v|."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R
import media_reference as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


@pytest.fixture(params=["rows", "planned", "stream", None], autouse=True)
def form(request, monkeypatch):
    if request.param:
        monkeypatch.setenv("TTPA_CROSS_FORM", request.param)
    return request.param


def _check(out, q, k, v, table, lens, scale):
    want, spread = M.cross(q, k, v, table, lens, scale)
    err = (out.cpu().double() - want).abs()
    tol = 2.0**-8 * want.abs() + (2 * 2.0**-8 * 1.005 + 6e-4) * spread + 1e-30
    assert bool((err <= tol).all()), ((~(err <= tol)).nonzero()[:4].tolist(), float((err / tol).nan_to_num(1e9).max()))


def _inputs(g, users, hq, hkv, s, d, bs, lens, width):
    """Elements and scales, and the values that they stand for; behind the last key NaN, and scales that are anything where a block holds no key."""
    nb = users * width + 2
    table = (torch.randperm(nb - 1, generator=g)[: users * width] + 1).view(users, width).int()
    elements = [torch.randn(nb, hkv, bs, d, generator=g).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ldexp(torch.ones(nb, hkv), torch.randint(-8, -4, (nb, hkv), generator=g)) for _ in range(2)]
    values = [(R.values(e) * sc.double()[..., None, None]).to(torch.bfloat16) for e, sc in zip(elements, scales)]
    for u, n in enumerate(lens):
        for c in range(width):
            if n < c * bs + bs:
                for e in elements:
                    e.view(torch.uint8)[int(table[u, c]), :, max(0, n - c * bs) :] = 0x7F
            if n <= c * bs:
                for i, sc in enumerate(scales):
                    sc[int(table[u, c])] = (float("nan"), float("inf"), 0.0, -1.0)[(c + i) % 4]
    q = torch.randn(users, s, hq, d, generator=g).to(torch.bfloat16).transpose(1, 2)
    return q, elements, scales, values, table


def _run(q, elements, scales, table, lens, **kw):
    return torch.ops.tt.paged_fp8_cross_attention(q.cuda(), *(e.cuda() for e in elements), *(s.cuda() for s in scales), table.cuda(),
                                                  torch.as_tensor(lens).cuda(), **kw)


@pytest.mark.parametrize("d, bs", [(64, 32), (64, 64), (128, 32), (128, 96), (256, 32), (256, 64)])
@pytest.mark.parametrize("hkv, grp, s", [(2, 4, 1), (1, 16, 1), (2, 4, 5), (1, 40, 1), (2, 2, 33), (1, 1, 300)])
@pytest.mark.parametrize("lens", [(0, 1, 31, 32, 33, 64), (200, 0, 127, 65), (900,)])
def test_lengths(d, bs, hkv, grp, s, lens):
    g = torch.Generator().manual_seed(d + bs + s + grp)
    q, elements, scales, values, table = _inputs(g, len(lens), hkv * grp, hkv, s, d, bs, lens, -(-max(lens) // bs) + 1)
    for kw in ({}, {"most_keys": max(lens), "scale": 0.3 * d**-0.5}):
        out = _run(q, elements, scales, table, lens, **kw)
        assert out.stride() == q.stride()
        _check(out, q, *values, table, lens, kw.get("scale", d**-0.5))


@pytest.mark.parametrize("d, hq, hkv, s", [(128, 8, 2, 1), (64, 16, 2, 8), (256, 4, 2, 3)])
def test_many_users_of_all_lengths(d, hq, hkv, s):
    g = torch.Generator().manual_seed(d)
    lens = torch.randint(0, 70, (90,), generator=g)
    lens[40] = 2500
    q, elements, scales, values, table = _inputs(g, 90, hq, hkv, s, d, 32, lens.tolist(), 79)
    _check(_run(q, elements, scales, table, lens), q, *values, table, lens, d**-0.5)


@pytest.mark.parametrize("s", [1, 40])
def test_pages_outside_and_outputs_in_place(s):
    g = torch.Generator().manual_seed(s)
    lens = (70, 300)
    q, elements, scales, values, table = _inputs(g, 2, 8, 2, s, 128, 32, lens, 10)
    table[1, 3], table[0, 1] = -5, 10**6  # (read block 0)
    want = _run(q, elements, scales, table, lens)
    _check(want, q, *values, table, lens, 128**-0.5)
    own = q.cuda().clone(memory_format=torch.preserve_format)
    torch.ops.tt.paged_fp8_cross_attention_out(own, *(e.cuda() for e in elements), *(x.cuda() for x in scales), table.cuda(), torch.tensor(lens).cuda(), own)
    assert torch.equal(own, want)


def test_refusals():
    k = torch.zeros(4, 2, 32, 64, device="cuda").to(torch.float8_e4m3fn)
    ks = torch.ones(4, 2, device="cuda")
    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    op = torch.ops.tt.paged_fp8_cross_attention
    for args in [(q, k.float(), k, ks, ks, table, lens), (q, k, k[:2], ks, ks, table, lens), (q, k, k, ks[:2], ks, table, lens), (q, k, k, ks.double(), ks, table, lens),
                 (q[:, :3], k, k, ks, ks, table, lens), (q, k, k, ks, ks, table, lens.float()), (q, k, k, ks, ks, table, lens, -1.0)]:
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(NotImplementedError):
        op(q.clone().requires_grad_(), k, k, ks, ks, table, lens)
    small = torch.zeros(4, 2, 16, 64, device="cuda").to(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        op(q, small, small, ks, ks, table, lens)


@pytest.mark.parametrize("tokens", [1, 80])
@pytest.mark.parametrize("bounds", [False, True])
def test_a_layer_of_the_backend(tokens, bounds):
    """States written by a prompt's pass, read by it and by a step; captured and replayed for other lengths."""
    import numpy as np

    from tt_xla_amd import CrossMetadataBuilder, TTAttentionBackendImpl, fp8_ops

    g = torch.Generator().manual_seed(tokens)
    impl = TTAttentionBackendImpl(8, 128, 128**-0.5, 2, kv_cache_dtype="fp8_e4m3", attn_type="encoder_decoder")
    k_cache, k_scales = fp8_ops.fp8_empty_cache(20, 2, 32, 128, device="cuda")
    v_cache, v_scales = fp8_ops.fp8_empty_cache(20, 2, 32, 128, device="cuda")
    cache = [k_cache, v_cache, k_scales, v_scales] + ([fp8_ops.fp8_empty_key_bounds(20, 2, 128, device="cuda")] if bounds else [])
    builder = CrossMetadataBuilder(32, 5, device="cuda")
    blocks = (torch.randperm(19, generator=g)[:15] + 1).view(3, 5).numpy()
    lens = [70, 0, 130]
    k, v = (torch.randn(2, 130, 2, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(3, tokens, 8, 128, generator=g).to(torch.bfloat16)
    out = torch.empty(3 * tokens, 1024, dtype=torch.bfloat16, device="cuda")
    md = builder.prepare(blocks, np.array(lens), new_rows=[0, 2])
    impl.forward(None, q.reshape(3 * tokens, -1).cuda(), k.reshape(260, -1).cuda(), v.reshape(260, -1).cuda(), cache, md, output=out)

    def check(lens):
        values = [(R.values(e.cpu()) * s.cpu().double()[..., None, None]).to(torch.bfloat16) for e, s in ((k_cache, k_scales), (v_cache, v_scales))]
        _check(out.view(3, tokens, 8, 128).transpose(1, 2), q.transpose(1, 2), *values, torch.from_numpy(blocks).int(), lens, 128**-0.5)

    check(lens)
    run = lambda: impl.forward(None, q_on, None, None, cache, md, output=out)  # noqa: E731
    q_on = q.reshape(3 * tokens, -1).cuda()
    md = builder.prepare(blocks, np.array(lens))
    run()
    check(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for now in ([70, 0, 130], [3, 0, 1], [64, 0, 97]):
        builder.prepare(blocks, np.array(now))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(now)
