"""A small model of pictures beside text, as it would be served: keys and queries rotated by time, height and width, prompts into a paged cache, attention to
an encoder's states in a second one, forks of requests with copies of the pages that they write, drafted tokens of which some are kept, and pages that move
together; ``tt_xla_amd``'s backend, ``CachePages`` and the operators in turn, every result against softmax in 64 bits over the tokens' own history.

Tolerance: a weight is rounded to bfloat16 (2^-8 of it), its normaliser is a sum of rounded or of unrounded ones, the result is rounded once more, and the scores'
sums and the exponential add less than 6e-4 of a weight, twice: 2^-8 |out| + (2 * 2^-8 * 1.005 + 6e-4) sum p |v|.  A rotated row: see ``test_gpu_rope_axes.py``: 2^-8 of
the value and 2^-19 of the pair's length for the products in float32."""

import numpy as np
import pytest
import torch

import __graft_entry__ as entry
import media_reference as M

pytestmark = pytest.mark.gpu

HQ, HKV, BS, WIDTH, ENC_WIDTH = 8, 2, 32, 8, 5


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


def _bf(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16)


def _close(got, want, spread):
    err = (got.double() - want).abs()
    tol = 2.0**-8 * want.abs() + (2 * 2.0**-8 * 1.005 + 6e-4) * spread + 1e-30
    assert bool((err <= tol).all()), float((err / tol).nan_to_num(1e9).max())


def _attend(q, k, v, scale, causal_from=None):
    """q [tokens, HQ, d] over k, v [keys, HKV, d] -> (out, spread) float64; causal_from: the position of the first row."""
    g = HQ // HKV
    k, v = (x.double().repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2).contiguous() * scale
    if causal_from is not None:
        s.masked_fill_(torch.arange(k.shape[1])[None] > causal_from + torch.arange(q.shape[0])[:, None], float("-inf"))
    p = torch.softmax(s, -1) if k.shape[1] else s
    return (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)


class Model:
    """Two layers, one of them cross attention, over the pages of two caches."""

    def __init__(self, d, seed):
        from tt_xla_amd import CachePages, CrossMetadataBuilder, TTAttentionBackendImpl
        from tt_xla_amd.media_ops import rope_pair_axes

        self.g, self.d, self.scale = torch.Generator().manual_seed(seed), d, d**-0.5
        self.pages, self.enc_pages = CachePages(40, BS), CachePages(24, BS)
        cache = lambda nb: [_bf(self.g, nb, HKV, BS, d).mul_(100).cuda() for _ in range(2)]  # noqa: E731
        self.kv, self.enc = {"self": cache(40), "other": cache(40)}, {"cross": cache(24)}
        self.layer = TTAttentionBackendImpl(HQ, d, self.scale, HKV)
        self.cross = TTAttentionBackendImpl(HQ, d, self.scale, HKV, attn_type="encoder_decoder")
        self.builder = CrossMetadataBuilder(BS, ENC_WIDTH, device="cuda")
        angle = torch.arange(600)[:, None] * 10000.0 ** (-torch.arange(d // 2) / (d // 2))
        self.table = torch.cat([angle.cos(), angle.sin()], 1)
        self.axes = rope_pair_axes([d // 8 * 2, d // 8, d // 8])
        self.w = _bf(self.g, d)
        self.k, self.v, self.ek, self.ev = {}, {}, {}, {}  # of every request: what its tokens' keys and values are

    def turn(self, q, k, positions):
        """Rotated on the GPU, as bfloat16 on the host."""
        on = torch.ops.tt.qk_norm_rope_axes(q.cuda(), k.cuda(), self.table.cuda(), positions.int().cuda(), self.axes.cuda(), self.w.cuda(), self.w.cuda())
        for got, x in zip(on, (q, k)):
            want = M.turn_axes(x, self.w, self.table, positions, self.axes, 1e-6, False)
            plain = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6) * self.w.double()
            norm = torch.hypot(plain[..., : self.d // 2], plain[..., self.d // 2 :]).repeat(1, 1, 2)
            assert bool(((got.cpu().double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-19 * norm).all())
        return [x.cpu() for x in on]

    def rows(self, n):
        return _bf(self.g, n, HQ, self.d), _bf(self.g, n, HKV, self.d), _bf(self.g, n, HKV, self.d)

    def copy(self, pairs):
        from tt_xla_amd import copy_cache_blocks

        copy_cache_blocks(self.kv, pairs)

    def pass_(self, names, n, decode):
        """n new tokens for every request (their pages are there): through the self attention layer, and their rows against the encoder's states.  Prompts are padded
        to whole blocks of 32 rows, as that layer takes them."""
        from tt_xla_amd import TTMetadata

        real, n = n, n if decode else -(-n // 32) * 32

        starts = [len(self.k[s]) if s in self.k else 0 for s in names]
        q, k, v = self.rows(len(names) * n)
        at = torch.cat([torch.arange(n) + s for s in starts])
        q, k = self.turn(q, k, torch.stack([at, at // 7, at % 7]))
        q, k, v = (x.unflatten(0, (len(names), n)) for x in (q, k, v))
        for i, s in enumerate(names):
            self.k[s], self.v[s] = (torch.cat([old[s], new[i]]) if s in old else new[i, :real] for old, new in ((self.k, k), (self.v, v)))
        table = self.pages.table(names, WIDTH).cuda()
        position = torch.tensor(starts, dtype=torch.int32, device="cuda")
        md = TTMetadata(cache_position=position if decode else None, page_table=table, num_users=len(names), is_causal=True,
                        batch_idx=torch.arange(len(names), dtype=torch.int32, device="cuda"))
        flat = lambda x: x.reshape(len(names) * n, -1).cuda()  # noqa: E731
        out = torch.empty(len(names) * n, HQ * self.d, dtype=torch.bfloat16, device="cuda")
        for cache in self.kv.values():
            self.layer.forward(None, flat(q), flat(k), flat(v), cache, md, output=out)
            for i, s in enumerate(names):
                _close(out.cpu().view(len(names), n, HQ, self.d)[i, :real], *_attend(q[i, :real], self.k[s], self.v[s], self.scale, starts[i]))
        self.see(names, flat(q), q)

    def see(self, names, q_flat, q, new=(), states=None):
        n = q.shape[1]
        lens = np.array([len(self.ek[s]) for s in names])
        md = self.builder.prepare(self.enc_pages.table(names, ENC_WIDTH).numpy(), lens, new, target_num_reqs=len(names))
        out = torch.full((len(names) * n, HQ * self.d), float("nan"), dtype=torch.bfloat16, device="cuda")
        k, v = states if states else (None, None)
        self.cross.forward(None, q_flat, k, v, self.enc["cross"], md, output=out)
        for i, s in enumerate(names):
            _close(out.cpu().view(len(names), n, HQ, self.d)[i], *_attend(q[i], self.ek[s], self.ev[s], self.scale))
        return out

    def encode(self, names, lens):
        """Encoder states of some requests in one pass, padded with what must not be used; a look at them with three tokens each."""
        fill = [i for i, n in enumerate(lens) if n]
        most = max(lens)
        k, v = (torch.full((len(fill), most, HKV, self.d), float("nan"), dtype=torch.bfloat16) for _ in range(2))
        for s, n in zip(names, lens):
            self.enc_pages.add(s, n)
            self.ek[s], self.ev[s] = _bf(self.g, n, HKV, self.d), _bf(self.g, n, HKV, self.d)
        for row, i in enumerate(fill):
            k[row, : lens[i]], v[row, : lens[i]] = self.ek[names[i]], self.ev[names[i]]
        q = _bf(self.g, len(names), 3, HQ, self.d)
        self.see(names, q.reshape(len(names) * 3, -1).cuda(), q, fill, [x.reshape(-1, HKV * self.d).cuda() for x in (k, v)])

    def keep(self, name, first, chosen):
        """Of the tokens from `first` on those of `chosen` stay."""
        self.copy(self.pages.own(name, first))
        kept = torch.tensor([chosen], dtype=torch.int32, device="cuda")
        tensors = [t for c in self.kv.values() for t in c]
        torch.ops.tt.keep_cache_tokens_(tensors, self.pages.table([name], WIDTH).cuda(), kept, torch.tensor([len(chosen)], device="cuda"),
                                        torch.tensor([first], device="cuda"))
        self.pages.truncate(name, first + len(chosen))
        for x in (self.k, self.v):
            x[name] = torch.cat([x[name][:first], x[name][chosen]])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_served_model(d):
    m = Model(d, d)
    m.encode(["a", "b", "c"], [70, 0, 33])
    for s in "abc":
        m.pages.add(s, 45)
    m.pass_(list("abc"), 45, decode=False)
    # a second answer to request a, on the same pages and states
    m.pages.fork("a", "a2")
    m.enc_pages.fork("a", "a2")
    for x in (m.k, m.v, m.ek, m.ev):
        x["a2"] = x["a"]
    for _ in range(3):
        pairs = [p for s in ("a", "a2", "b") for p in m.pages.extend(s, 1)]
        m.copy(pairs)
        m.pass_(["a", "a2", "b"], 1, decode=True)
    assert m.pages.pages("a")[0] == m.pages.pages("a2")[0] and m.pages.pages("a")[1] != m.pages.pages("a2")[1]
    # a tree of drafts: twenty tokens behind request c's, across a page's end, of which seven stay
    first = m.pages.length("c")
    for _ in range(20):
        m.copy(m.pages.extend("c", 1))
        m.pass_(["c"], 1, decode=True)
    m.keep("c", first, [first + i for i in (0, 3, 4, 9, 12, 13, 19)])
    m.copy(m.pages.extend("c", 1) + m.pages.extend("a2", 1))
    m.pass_(["c", "a2"], 1, decode=True)
    # tokens leave from the middle of what a and a2 share
    m.keep("a", 5, list(range(9, 48, 2)))
    m.copy(m.pages.extend("a2", 1) + m.pages.extend("a", 1))
    m.pass_(["a2", "a"], 1, decode=True)
    # requests end, their pages are free, the others' move together
    for p in (m.pages, m.enc_pages):
        p.free("b"), p.free("a")
    m.copy(m.pages.compact())
    from tt_xla_amd import copy_cache_blocks

    copy_cache_blocks(m.enc, m.enc_pages.compact())
    m.copy([p for s in ("a2", "c") for p in m.pages.extend(s, 1)])
    m.pass_(["a2", "c"], 1, decode=True)
    m.pages.add("e", 33)
    m.encode(["e"], [150])
    m.pass_(["e"], 33, decode=False)
    m.copy([p for s in ("e", "c") for p in m.pages.extend(s, 1)])
    m.pass_(["e", "c"], 1, decode=True)


@pytest.mark.parametrize("tokens", [1, 4, 70])
def test_a_captured_pass_for_other_lengths(tokens):
    """The pass is captured with one metadata and replayed for others of the same buffers: it has to have room for the longest."""
    m = Model(128, 5)
    m.encode(["a", "b", "c"], [3, 2, 1])
    q = _bf(m.g, 3, tokens, HQ, 128)
    flat, out = q.reshape(3 * tokens, -1).cuda(), torch.empty(3 * tokens, HQ * 128, dtype=torch.bfloat16, device="cuda")
    names = list("abc")
    md = m.builder.prepare(m.enc_pages.table(names, ENC_WIDTH).numpy(), np.array([3, 2, 1]))
    run = lambda: m.cross.forward(None, flat, None, None, m.enc["cross"], md, output=out)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lens in ([3, 2, 1], [160, 0, 33], [0, 0, 0], [64, 159, 5]):
        for s, n in zip(names, lens):
            m.enc_pages.free(s)
            del m.ek[s], m.ev[s]
        m.encode(names, lens) if any(lens) else [(m.enc_pages.add(s, 0), m.ek.update({s: _bf(m.g, 0, HKV, 128)}), m.ev.update({s: _bf(m.g, 0, HKV, 128)})) for s in names]
        m.builder.prepare(m.enc_pages.table(names, ENC_WIDTH).numpy(), np.array(lens))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(names):
            _close(out.cpu().view(3, tokens, HQ, 128)[i], *_attend(q[i], m.ek[s], m.ev[s], m.scale))


@pytest.mark.parametrize("how", ["float32", "unaligned", "column"])
def test_outputs_that_the_kernel_cannot_write(how):
    m = Model(64, 9)
    m.encode(["a", "b"], [40, 7])
    md = m.builder.prepare(m.enc_pages.table(["a", "b"], ENC_WIDTH).numpy(), np.array([40, 7]))
    q = _bf(m.g, 2, 5, HQ, 64)
    want = torch.empty(10, HQ * 64, dtype=torch.bfloat16, device="cuda")
    out = {"float32": torch.empty(10, HQ * 64, device="cuda"), "unaligned": torch.empty(10 * HQ * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(10, -1),
           "column": torch.empty(10, 2, HQ * 64, dtype=torch.bfloat16, device="cuda")[:, 1]}[how]
    for o in (want, out):
        m.cross.forward(None, q.reshape(10, -1).cuda(), None, None, m.enc["cross"], md, output=o)
    assert torch.equal(out.to(torch.bfloat16), want)


@pytest.mark.parametrize("keys", [1, 50])
def test_without_a_cache_the_states_of_the_pass_are_attended(keys):
    from tt_xla_amd import TTMetadata

    m = Model(128, 3)
    q, k, v = _bf(m.g, 2, 6, HQ, 128), _bf(m.g, 2, keys, HKV, 128), _bf(m.g, 2, keys, HKV, 128)
    md = TTMetadata(cache_position=None, page_table=torch.zeros(2, 1, dtype=torch.int32, device="cuda"), num_users=2)
    out = torch.empty(12, HQ * 128, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.bfloat16, device="cuda")
    m.cross.forward(None, q.reshape(12, -1).cuda(), k.reshape(2 * keys, -1).cuda(), v.reshape(2 * keys, -1).cuda(), [none, none], md, output=out)
    for i in range(2):
        _close(out.cpu().view(2, 6, HQ, 128)[i], *_attend(q[i], k[i], v[i], m.scale))
