"""Rotation by several axes, cross attention and moves inside caches on the host: schemas, what the C entry points refuse before any launch, what a
cross attention layer refuses, and the axes of pairs."""

import pytest
import torch

import __graft_entry__ as entry

ROPE = ("Tensor cos_sin, Tensor positions, Tensor pair_axes, Tensor? q_weight=None, Tensor? k_weight=None, float eps=9.9999999999999995e-07, "
        "bool interleaved=False")
CROSS = "Tensor query, Tensor key, Tensor value, Tensor page_table, Tensor encoder_lens"
SCHEMAS = {
    "qk_norm_rope_axes": f"tt::qk_norm_rope_axes(Tensor query, Tensor key, {ROPE}) -> (Tensor, Tensor)",
    "qk_norm_rope_axes_": f"tt::qk_norm_rope_axes_(Tensor(a!) query, Tensor(b!) key, {ROPE}) -> ()",
    "paged_cross_attention": f"tt::paged_cross_attention({CROSS}, float? scale=None, int most_keys=0) -> Tensor",
    "paged_cross_attention_out": f"tt::paged_cross_attention_out({CROSS}, Tensor(a!) out, float? scale=None, int most_keys=0) -> ()",
    "paged_fp8_cross_attention": "tt::paged_fp8_cross_attention(Tensor query, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, Tensor page_table, "
                                 "Tensor encoder_lens, float? scale=None, int most_keys=0) -> Tensor",
    "copy_cache_blocks_": "tt::copy_cache_blocks_(Tensor(a!)[] caches, Tensor source_blocks, Tensor target_blocks) -> ()",
    "keep_cache_tokens_": "tt::keep_cache_tokens_(Tensor(a!)[] caches, Tensor page_table, Tensor kept, Tensor kept_lens, Tensor? first=None) -> ()",
}


@pytest.fixture(scope="module")
def lib():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401
    from tt_xla_amd import _native

    return _native.lib()


@pytest.mark.parametrize("name", sorted(SCHEMAS))
def test_schema(lib, name):
    assert str(getattr(torch.ops.tt, name).default._schema).replace("eps=1e-06", "eps=9.9999999999999995e-07") == SCHEMAS[name]


def test_cpu_tensors_are_refused(lib):
    z, ids = torch.zeros(2, 1, 32, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: torch.ops.tt.paged_cross_attention(z[:1, :, :1], z, z, ids[None], ids),
                 lambda: torch.ops.tt.qk_norm_rope_axes(x, x, torch.zeros(4, 64), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(32, dtype=torch.int32)),
                 lambda: torch.ops.tt.copy_cache_blocks_([z], ids, ids), lambda: torch.ops.tt.keep_cache_tokens_([z], ids[None], ids[None], ids)):
        with pytest.raises(NotImplementedError):
            call()


def test_fakes_have_the_results_shapes(lib):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = torch.empty(5, 8, 128, dtype=torch.bfloat16), torch.empty(5, 2, 128, dtype=torch.bfloat16)
        out = torch.ops.tt.qk_norm_rope_axes(q, k, torch.empty(9, 128), torch.empty(3, 5, dtype=torch.int32), torch.empty(64, dtype=torch.int32))
        assert [o.shape for o in out] == [q.shape, k.shape]
        z, x = torch.empty(4, 2, 32, 64, dtype=torch.bfloat16), torch.empty(3, 8, 7, 64, dtype=torch.bfloat16)
        pt, lens = torch.empty(3, 2, dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        assert torch.ops.tt.paged_cross_attention(x, z, z, pt, lens).shape == x.shape
        assert torch.ops.tt.paged_cross_attention_out(x, z, z, pt, lens, x) is None
        assert torch.ops.tt.copy_cache_blocks_([z], lens, lens) is None and torch.ops.tt.keep_cache_tokens_([z], pt, pt, lens) is None


# arguments that are in order, by name; pointers are aligned numbers that nothing follows (every call below is refused first)
def _rope(lib, q=16, strides=512, eps=1e-6, tokens=4, heads=4, d=128, rotary=128, axes=3, pair_axes=16, row_stride=128, most=100):
    return lib.ttpa_qk_norm_rope_axes(16, strides, 128, 16, strides, 128, q, strides, 128, 16, strides, 128, 16, 1, row_stride, most, 16, 0, 4, axes,
                                      pair_axes, None, None, 0, eps, tokens, heads, 2, d, rotary, 0, None)


def _cross(lib, q=16, lens=16, users=2, hq=8, hkv=2, s=3, d=128, bs=64, w=4, nb=8, scale=1.0, most=0, stride=1024, ws=256, ws_bytes=1 << 40):
    return lib.ttpa_paged_cross_attention(16, 1 << 16, 128, 1024, q, 1 << 16, 128, stride, 16, 16, 16, 4, lens, 0, users, hq, hkv, s, d, bs, w, nb,
                                          scale, most, ws, ws_bytes, None)


def _cross8(lib, q=16, scales=16, users=2, hq=8, hkv=2, s=3, d=128, bs=64, w=4, nb=8, scale=1.0, most=0, ws=256, ws_bytes=1 << 40):
    return lib.ttpa_paged_fp8_cross_attention(16, 1 << 16, 128, 1024, q, 1 << 16, 128, 1024, 16, 16, scales, 16, 16, 4, 16, 0, users, hq, hkv, s, d, bs, w, nb,
                                              scale, most, ws, ws_bytes, None)


def _some(n=1, p=256):
    import ctypes

    return (ctypes.c_void_p * max(n, 1))(*([p] * n))


def _copy(lib, caches=256, n=1, bytes_=64, source=16, pairs=2, nb=8):
    import ctypes

    sizes = None if bytes_ is None else (ctypes.c_int64 * max(n, 1))(*([bytes_] * n))
    return lib.ttpa_copy_cache_blocks(_some(n, caches) if caches != "none" else None, sizes, n, source, 16, pairs, nb, None)


def _keep(lib, caches=256, n=1, pt=16, users=2, most=4, heads=2, row=128, bs=32, w=4, nb=8):
    return lib.ttpa_keep_cache_tokens(_some(n, caches), n, pt, 4, 16, 4, 16, None, users, most, heads, row, bs, w, nb, None)


@pytest.mark.parametrize("call, wrong, status, says", [
    (_rope, dict(q=None), -1, b"null"), (_rope, dict(strides=516), -1, b"strides"), (_rope, dict(eps=-1.0), -1, b"eps"),
    (_rope, dict(tokens=-1), -1, b"dimension"), (_rope, dict(heads=0), -1, b"dimension"), (_rope, dict(d=96), -2, b"head_size"),
    (_rope, dict(rotary=24), -1, b"rotary"), (_rope, dict(axes=0), -2, b"axes"), (_rope, dict(axes=100), -2, b"axes"), (_rope, dict(pair_axes=None), -1, b"pair_axes"),
    (_rope, dict(pair_axes=20), -1, b"pair_axes"), (_rope, dict(most=1 << 40), -1, b"angles"), (_rope, dict(row_stride=-8), -1, b"angles"),
    (_cross, dict(q=None), -1, b"null"), (_cross, dict(lens=None), -1, b"null"), (_cross, dict(users=-1), -1, b"dimension"), (_cross, dict(hq=9), -1, b"divisible"),
    (_cross, dict(d=96), -2, b"head_size"), (_cross, dict(bs=48), -2, b"block_size"), (_cross, dict(bs=8192), -2, b"block_size"),
    (_cross, dict(scale=0.0), -1, b"scale"), (_cross, dict(scale=-1.0), -1, b"scale"), (_cross, dict(most=-1), -1, b"most_keys"), (_cross, dict(w=1 << 26), -1, b"too many keys"),
    (_cross, dict(q=24), -1, b"aligned"), (_cross, dict(stride=1028), -1, b"strides"), (_cross, dict(ws_bytes=0, users=1, w=400), -3, b"workspace"),
    (_cross8, dict(q=None), -1, b"null"), (_cross8, dict(scales=None), -1, b"null"), (_cross8, dict(hq=9), -1, b"divisible"), (_cross8, dict(d=96), -2, b"head_size"),
    (_cross8, dict(bs=16), -2, b"block_size"), (_cross8, dict(scale=0.0), -1, b"scale"), (_cross8, dict(ws_bytes=0, users=1, w=400), -3, b"workspace"),
    (_cross8, dict(ws_bytes=0, users=8, s=600, w=100, nb=1000), -3, b"workspace"),
    (_copy, dict(caches=None), -1, b"null"), (_copy, dict(caches="none"), -1, b"null"), (_copy, dict(source=None), -1, b"null"), (_copy, dict(bytes_=0), -1, b"bytes"), (_copy, dict(bytes_=1 << 31), -1, b"bytes"), (_copy, dict(bytes_=None), -1, b"null"),
    (_copy, dict(pairs=-1), -1, b"dimension"), (_copy, dict(nb=0), -1, b"dimension"), (_copy, dict(n=-1), -1, b"null"),
    (_keep, dict(caches=None), -1, b"null"), (_keep, dict(pt=None), -1, b"null"), (_keep, dict(users=-1), -1, b"dimension"), (_keep, dict(row=24), -2, b"multiples of 16"),
    (_keep, dict(caches=264), -1, b"aligned"), (_keep, dict(w=1 << 26), -1, b"too many tokens"), (_keep, dict(heads=1 << 24), -1, b"too many rows"),
])
def test_c_refusals(lib, call, wrong, status, says):
    assert call(lib, **wrong) == status
    assert says in lib.ttpa_last_error(), lib.ttpa_last_error()


def test_c_calls_of_nothing(lib):
    assert _rope(lib, tokens=0) == 0 and _cross(lib, users=0) == 0 and _cross(lib, s=0) == 0
    assert _copy(lib, pairs=0) == 0 and _copy(lib, n=0) == 0 and _keep(lib, users=0) == 0 and _keep(lib, most=0) == 0 and _keep(lib, n=0) == 0


def test_axes_of_pairs(lib):
    from tt_xla_amd.media_ops import rope_pair_axes

    assert rope_pair_axes([2, 3, 1]).tolist() == [0, 0, 1, 1, 1, 2]
    assert rope_pair_axes([4, 2, 2], alternating=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rope_pair_axes([3], alternating=True).tolist() == [0, 0, 0] and rope_pair_axes([0, 2]).tolist() == [1, 1]
    pairs = rope_pair_axes([24, 20, 20], alternating=True)
    assert [int((pairs == a).sum()) for a in range(3)] == [24, 20, 20] and pairs.dtype == torch.int32
    for wrong, turns in (([], False), ([-1, 3], False), ([0, 0], False), ([1, 4], True)):
        with pytest.raises(ValueError):
            rope_pair_axes(wrong, turns)


# ---- a cross attention layer ------------------------------------------------------------------------
def _layer(**kw):
    from tt_xla_amd import TTAttentionBackendImpl

    return TTAttentionBackendImpl(**{**dict(num_heads=8, head_size=64, scale=0.125, num_kv_heads=2, attn_type="encoder_decoder"), **kw})


@pytest.mark.parametrize("wrong", [dict(sliding_window=64), dict(sinks=torch.zeros(8)), dict(sparse_kept_blocks=4), dict(functional_cache_ops=True),
                                   dict(kv_cache_dtype="bfp_bf8"), dict(head_size=96)])
def test_what_a_cross_attention_layer_is_not_built_with(lib, wrong):
    with pytest.raises(NotImplementedError, match="cross attention"):
        _layer(**wrong)


def test_what_a_cross_attention_pass_refuses_before_it_writes(lib):
    from tt_xla_amd import TTMetadata

    z = torch.zeros(4, 2, 32, 64, dtype=torch.bfloat16)
    x, kv = torch.zeros(2, 512, dtype=torch.bfloat16), torch.zeros(64, 128, dtype=torch.bfloat16)
    ids = torch.zeros(2, 2, dtype=torch.int32)
    one = dict(page_table=ids, num_users=2, batch_idx=ids[0], encoder_lens=ids[0])

    def run(error, says, key=kv, value=kv, cache=(z, z), **md):
        with pytest.raises(error, match=says):
            _layer().forward(None, x, key, value, cache, TTMetadata(cache_position=None, **{**one, **md}), output=torch.empty_like(x))

    run(NotImplementedError, "masks", attn_mask=torch.zeros(1, 1, 2, 64))
    run(ValueError, "or neither", key=None)
    run(ValueError, "encoder_lens", encoder_lens=None)
    run(AssertionError, "num_users", num_users=None)
    run(AssertionError, "batch_idx", batch_idx=None)
    run(ValueError, "divisible", num_users=3)
    for cache in ((z.float(), z.float()), (z.view(torch.uint8),) * 2, (z, z, z), z, (z[:, :, :16],) * 2):
        run(NotImplementedError, "bfloat16 caches", cache=cache)
    for cache in ((z[:0], z[:0]), (), None):
        run(ValueError, "without a cache", key=None, value=None, cache=cache)
    assert not z.any()


def test_metadata_of_cross_attention(lib):
    import numpy as np

    from tt_xla_amd import CrossMetadataBuilder

    b = CrossMetadataBuilder(32, 4)
    blocks = np.arange(1, 13, dtype=np.int64).reshape(3, 4)
    md = b.prepare(blocks, np.array([33, 0, 128]), new_rows=[0, 2], target_num_reqs=4)
    assert md.page_table.tolist() == [[1, 2, -1, -1], [-1] * 4, [9, 10, 11, 12], [-1] * 4] and md.fill_page_table is md.page_table
    assert md.encoder_lens.tolist() == [33, 0, 128, 0] and md.most_encoder_len == 128 and md.batch_idx.tolist() == [0, 2] and md.num_users == 4
    again = b.prepare(blocks[:1], np.array([5]), target_num_reqs=4)
    assert again.page_table is md.page_table and again.encoder_lens.tolist() == [5, 0, 0, 0] and again.batch_idx is None
    for wrong in (dict(encoder_lens=np.array([129])), dict(encoder_lens=np.array([-1])), dict(encoder_lens=np.array([1]), new_rows=[1])):
        with pytest.raises(ValueError):
            b.prepare(blocks, **wrong)
