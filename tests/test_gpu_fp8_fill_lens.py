"""Prompts and encoder states into the 8-bit cache with a length for every row of the page table (``tt::paged_fill_fp8_cache_.lens``): what lies behind a row's
length, whatever it is, has no part in a scale or in bounds and is not written.  Elements, scales and bounds are whole steps of exact numbers, so all of them are equal
to those of a fill with the rows cut to their lengths."""

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _noise(nb, hkv, bs, d, g, bounds=True):
    """A cache with anything in it."""
    e = [torch.randint(0, 256, (nb, hkv, bs, d), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn).cuda() for _ in range(2)]
    s = [torch.ldexp(torch.ones(nb, hkv), torch.randint(-12, 4, (nb, hkv), generator=g)).cuda() for _ in range(2)]
    return (*e, *s), torch.randn(nb, hkv, 2, d, generator=g).to(torch.bfloat16).cuda() if bounds else None


def _states(g, users, tokens, hkv, d, lens, padding):
    """[users, hkv, tokens, d] of one length each, with `padding` behind a user's own."""
    out = []
    for _ in range(2):
        x = (torch.randn(users, tokens, hkv, d, generator=g) * 2.0 ** torch.randint(-8, 8, (users, 1, hkv, 1), generator=g)).to(torch.bfloat16)
        for u, n in enumerate(lens):
            x[u, max(0, n) :] = padding * (1 - 2 * (torch.arange(d) % 2))
        out.append(x.transpose(1, 2))
    return out


# (head size and block size: 1, 2, 4 and 8 pieces of a wavefront, 4, 8 and 16 of a workgroup, blocks that are read twice)
FORMS = [(64, 16), (128, 16), (128, 32), (64, 64), (128, 64), (256, 64), (128, 256), (256, 512), (64, 4096)]


@pytest.mark.parametrize("d, bs", FORMS)
@pytest.mark.parametrize("padding", [1e4, float("nan"), float("inf")])
@pytest.mark.parametrize("bounds", [False, True])
def test_rows_behind_a_length_have_no_part(d, bs, padding, bounds):
    g = torch.Generator().manual_seed(d + bs)
    hkv, blocks = 3, 2
    tokens = blocks * bs - 1
    lens = [1, 0, bs - 1, bs, bs + 1, tokens, tokens + 99, -3]
    users = len(lens)
    nb = users * blocks + 2
    cache, b = _noise(nb, hkv, bs, d, g, bounds)
    table = torch.randperm(nb, generator=g)[: users * blocks].view(users, blocks).int()
    rows = torch.randperm(users, generator=g)
    k, v = _states(g, users, tokens, hkv, d, [lens[r] for r in rows], padding)
    want = R.Cache(*cache, b)
    for i, r in enumerate(rows.tolist()):
        n = min(max(lens[r], 0), tokens)
        want.fill(k[i : i + 1, :, :n], v[i : i + 1, :, :n], table, [r])
    for dtype in (torch.int32, torch.int64):
        torch.ops.tt.paged_fill_fp8_cache_.lens(*cache, k.cuda(), v.cuda(), table.cuda(), rows.cuda(), b, lens=torch.tensor(lens, dtype=dtype).cuda())
        assert want.differences(*cache, b) == {}


@pytest.mark.parametrize("d, bs", [(64, 16), (128, 64), (128, 256)])
def test_lengths_that_leave_nothing_out(d, bs):
    """The bytes of the fill without lengths, from lengths beyond the table and beyond 32 bits, too."""
    g = torch.Generator().manual_seed(d)
    one, b1 = _noise(20, 2, bs, d, g)
    two, b2 = [x.clone() for x in one], b1.clone()
    k, v = _states(g, 3, 2 * bs + 5, 2, d, [1 << 30] * 3, 0.0)
    k[1, 0, 0, 3], v[2, 1, bs, 0] = float("nan"), float("inf")
    table, rows = torch.arange(9, dtype=torch.int32).view(3, 3).cuda(), torch.tensor([2, 0, 1]).cuda()
    torch.ops.tt.paged_fill_fp8_cache_(*one, k.cuda(), v.cuda(), table, rows, b1)
    torch.ops.tt.paged_fill_fp8_cache_(*two, k.cuda(), v.cuda(), table, rows, b2, lens=torch.tensor([2 * bs + 5, 1 << 31, 1 << 45]).cuda())
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((*one, b1), (*two, b2)))


def test_refusals():
    g = torch.Generator().manual_seed(1)
    cache, b = _noise(4, 2, 32, 64, g)
    k = torch.zeros(2, 2, 40, 64, dtype=torch.bfloat16, device="cuda")
    table, rows = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.arange(2, device="cuda")
    before = [x.clone() for x in (*cache, b)]
    fill = torch.ops.tt.paged_fill_fp8_cache_.lens
    for lens in (rows[:1], rows.float(), rows[None]):
        with pytest.raises(ValueError):
            fill(*cache, k, k, table, rows, b, lens=lens)
    with pytest.raises(NotImplementedError):
        fill(*cache, k, k, table, rows, b, lens=rows.cpu())
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip((*cache, b), before))


@pytest.mark.parametrize("bounds", [False, True])
@pytest.mark.parametrize("bs", [32, 64])
def test_a_cross_attention_layer_does_not_look_at_padding(bounds, bs):
    """The cache of a layer of the backend, filled with states that are padded to one length with numbers far above them, is that of a fill with every user's own states; also where the pass
    is captured and replayed with other lengths."""
    from tt_xla_amd import CrossMetadataBuilder, TTAttentionBackendImpl

    g = torch.Generator().manual_seed(bs)
    hq, hkv, d, width = 8, 2, 128, 5
    impl = TTAttentionBackendImpl(hq, d, d**-0.5, hkv, kv_cache_dtype="fp8_e4m3", attn_type="encoder_decoder")
    cache, b = _noise(20, hkv, bs, d, g, bounds)
    kv = [*cache] + ([b] if bounds else [])
    builder = CrossMetadataBuilder(bs, width, device="cuda")
    blocks = (torch.randperm(19, generator=g)[:15] + 1).view(3, width).numpy()
    tokens = 130
    q = torch.randn(3, hq * d, generator=g).to(torch.bfloat16).cuda()
    k_on, v_on = (torch.empty(2 * tokens, hkv * d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.empty(3, hq * d, dtype=torch.bfloat16, device="cuda")

    def put(lens):
        """New states of users 0 and 2, and the cache that they should leave."""
        k, v = _states(g, 2, tokens, hkv, d, [lens[0], lens[2]], 1e4)
        for on, x in ((k_on, k), (v_on, v)):
            on.copy_(x.transpose(1, 2).reshape(2 * tokens, -1))
        want = R.Cache(*cache, b)
        table = builder.prepare(blocks, np.array(lens)).page_table.cpu()
        for i, u in enumerate((0, 2)):
            want.fill(k[i : i + 1, :, : lens[u]], v[i : i + 1, :, : lens[u]], table, [u])
        return want

    lens = [70, 0, 97]
    want = put(lens)
    md = builder.prepare(blocks, np.array(lens), new_rows=[0, 2])
    impl.forward(None, q, k_on, v_on, kv, md, output=out)
    assert want.differences(*cache, b) == {}
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        impl.forward(None, q, k_on, v_on, kv, md, output=out)
    for now in ([70, 0, 97], [1, 0, 130], [bs, 5, 0], [130, 0, 33]):
        want = put(now)
        graph.replay()
        torch.cuda.synchronize()
        assert want.differences(*cache, b) == {}


def test_a_fill_table_of_its_own_goes_without_lengths():
    """Later blocks of users whose first ones are there: the lengths belong to the page table, and all that comes is written."""
    from tt_xla_amd import TTAttentionBackendImpl, TTMetadata

    g = torch.Generator().manual_seed(5)
    impl = TTAttentionBackendImpl(4, 64, 0.125, 2, kv_cache_dtype="fp8_e4m3", attn_type="encoder_decoder")
    cache, b = _noise(12, 2, 32, 64, g)
    table, rest = torch.arange(10, dtype=torch.int32).view(2, 5), torch.tensor([[2, 3]], dtype=torch.int32)
    k, v = _states(g, 1, 40, 2, 64, [40], 0.0)
    want = R.Cache(*cache, b)
    want.fill(k, v, rest, [0])
    md = TTMetadata(page_table=table.cuda(), fill_page_table=rest.cuda(), batch_idx=torch.zeros(1, dtype=torch.int32, device="cuda"), num_users=2,
                    encoder_lens=torch.tensor([64 + 40, 10], dtype=torch.int32, device="cuda"))
    q, out = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 256, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, q, *(x.transpose(1, 2).reshape(40, -1).cuda() for x in (k, v)), [*cache, b], md, output=out)
    assert want.differences(*cache, b) == {}
