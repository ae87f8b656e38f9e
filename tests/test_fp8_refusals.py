"""The 8-bit cache on the host: schemas of its operators, and what its C entry points refuse before any launch."""

import pytest
import torch

import __graft_entry__ as entry
import fp8_reference as R

CACHE = "Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales"
WRITTEN = "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales"
SCHEMAS = {
    "qk_norm_rope": "tt::qk_norm_rope(Tensor query, Tensor key, Tensor cos_sin, Tensor positions, Tensor? q_weight=None, Tensor? k_weight=None, "
                    "float eps=9.9999999999999995e-07, bool interleaved=False) -> (Tensor, Tensor)",
    "paged_update_fp8_cache_": f"tt::paged_update_fp8_cache_({WRITTEN}, Tensor k_fill, Tensor v_fill, Tensor update_indices, Tensor page_table, "
                               "Tensor(e!)? key_bounds=None) -> ()",
    "paged_fill_fp8_cache_": f"tt::paged_fill_fp8_cache_({WRITTEN}, Tensor k_fill, Tensor v_fill, Tensor page_table, Tensor? batch_idx=None, "
                             "Tensor(e!)? key_bounds=None) -> ()",
    "paged_fp8_attention_decode": f"tt::paged_fp8_attention_decode(Tensor query, {CACHE}, Tensor page_table, Tensor cur_pos_tensor, "
                                  "Tensor? attention_sink=None, float? scale=None, int? sliding_window_size=None) -> Tensor",
    "paged_fp8_sparse_attention_decode": f"tt::paged_fp8_sparse_attention_decode(Tensor query, {CACHE}, Tensor key_bounds, Tensor page_table, "
                                         "Tensor cur_pos_tensor, int kept_blocks, float? scale=None) -> (Tensor, Tensor)",
    "chunked_fp8_attention": f"tt::chunked_fp8_attention(Tensor query, {CACHE}, Tensor page_table, Tensor chunk_start_idx_tensor, "
                             "float? scale=None, int most_keys=0) -> Tensor",
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
    z = torch.zeros(1, 1, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError):
        torch.ops.tt.paged_fp8_attention_decode(torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), z, z, torch.ones(1, 1), torch.ones(1, 1),
                                                torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


# arguments that are in order, by name; pointers are aligned numbers that nothing follows (every call below is refused first)
def _rope(lib, q=16, out=16, strides=512, eps=1e-6, tokens=4, heads=4, d=128, rotary=128):
    return lib.ttpa_qk_norm_rope(out, strides, 128, 16, strides, 128, q, strides, 128, 16, strides, 128, 16, 1, rotary, 100, 16, 0, None, None, 0,
                                 eps, tokens, heads, 2, d, rotary, 0, None)


def _decode(lib, q=16, scales=16, users=2, hq=8, hkv=2, d=128, bs=64, w=4, nb=8, window=0, ws=256, ws_bytes=1 << 30, q_stride=1024):
    return lib.ttpa_paged_fp8_decode(16, 1024, 128, q, q_stride, 128, 16, 16, scales, 16, 16, 4, 16, 0, users, hq, hkv, d, bs, w, nb, 1.0, window,
                                     None, ws, ws_bytes, None)


def _sparse(lib, bounds=16, kept=4, users=2, hq=8, hkv=2, d=128, bs=64, w=8, nb=8, ws=256, ws_bytes=1 << 40):
    return lib.ttpa_paged_fp8_sparse_decode(16, 128, 16, 16, 128, 16, 16, 16, 16, bounds, 16, 8, 16, 0, users, hq, hkv, d, bs, w, nb, kept, 1.0, ws,
                                            ws_bytes, None)


def _fill(lib, k=16, users=2, bidx=16, s=100, bs=64, d=128, w=4, token_stride=512):
    return lib.ttpa_paged_fill_fp8_cache(16, 16, 16, 16, None, k, 51200, 128, token_stride, 16, 51200, 128, 512, 16, 4, bidx, 0, users, 2, 2, s, bs,
                                         d, w, 8, None)


def _update(lib, k=16, users=2, d=128, bs=64, nb=8, head_stride=128):
    return lib.ttpa_paged_update_fp8_cache(16, 16, 16, 16, None, k, 512, head_stride, 16, 512, 128, 16, 0, 16, 4, users, 2, bs, d, 4, nb, None)


def _chunk(lib, q=16, bs=64, s=32, w=4, hq=8, ws=256, ws_bytes=1 << 40, most=0):
    return lib.ttpa_chunked_fp8_attention(16, 1 << 20, 1 << 15, 128, q, 1 << 20, 1 << 15, 128, 16, 16, 16, 16, 16, 4, 16, 1, hq, 2, s, 128, bs, w, 8,
                                          1.0, most, ws, ws_bytes, None)


@pytest.mark.parametrize("call, wrong, status, says", [
    (_rope, dict(q=None), -1, b"null"), (_rope, dict(out=8), -1, b"aligned"), (_rope, dict(strides=516), -1, b"strides"),
    (_rope, dict(eps=-1.0), -1, b"eps"), (_rope, dict(tokens=-1), -1, b"dimension"), (_rope, dict(heads=0), -1, b"dimension"),
    (_rope, dict(d=96, rotary=96), -2, b"head_size"), (_rope, dict(rotary=24), -1, b"rotary"), (_rope, dict(rotary=144), -1, b"rotary"),
    (_rope, dict(tokens=1 << 30), -1, b"too many"),
    (_decode, dict(q=None), -1, b"null"), (_decode, dict(scales=None), -1, b"null"), (_decode, dict(q=24), -1, b"aligned"),
    (_decode, dict(users=0), -1, b"dimension"), (_decode, dict(hq=7), -1, b"divisible"), (_decode, dict(hq=34), -2, b"up to 16"),
    (_decode, dict(d=96), -2, b"head_size"), (_decode, dict(bs=24), -2, b"block_size"), (_decode, dict(bs=8192), -2, b"block_size"),
    (_decode, dict(w=1 << 26), -1, b"page-table row"), (_decode, dict(nb=1 << 30), -1, b"num_blocks"), (_decode, dict(window=-1), -1, b"window"),
    (_decode, dict(users=2049), -2, b"users"), (_decode, dict(ws=None), -3, b"workspace"), (_decode, dict(ws=128), -3, b"workspace"),
    (_decode, dict(ws_bytes=1000), -3, b"workspace"), (_decode, dict(q_stride=1028), -1, b"strides"),
    (_sparse, dict(bounds=None), -1, b"bounds"), (_sparse, dict(kept=1), -1, b"kept_blocks"), (_sparse, dict(kept=1 << 26), -1, b"kept_blocks"),
    (_sparse, dict(ws=None), -3, b"workspace"), (_sparse, dict(ws_bytes=4096), -3, b"workspace"), (_sparse, dict(hq=9), -1, b"divisible"),
    (_sparse, dict(hq=8192, hkv=4096, nb=4), -2, b"KV heads"),
    (_fill, dict(k=None), -1, b"null"), (_fill, dict(k=8), -1, b"aligned"), (_fill, dict(bidx=None), -1, b"batch_idx"),
    (_fill, dict(s=257), -1, b"does not fit"), (_fill, dict(bs=40), -2, b"block_size"), (_fill, dict(users=-1), -1, b"dimension"),
    (_fill, dict(users=40000), -1, b"too many"), (_fill, dict(token_stride=500), -1, b"strides"),
    (_update, dict(k=None), -1, b"null"), (_update, dict(users=-1), -1, b"null"), (_update, dict(d=32), -2, b"head_size"),
    (_update, dict(nb=0), -1, b"dimension"), (_update, dict(head_stride=100), -1, b"strides"),
    (_chunk, dict(q=None), -1, b"null"), (_chunk, dict(bs=48), -2, b"multiple of 32"), (_chunk, dict(s=0), -1, b"dimension"),
    (_chunk, dict(hq=7), -1, b"divisible"), (_chunk, dict(ws=None), -3, b"workspace"), (_chunk, dict(ws_bytes=1000), -3, b"workspace"),
    (_chunk, dict(most=-1), -1, b"dimension"),
])
def test_refused_before_any_launch(lib, call, wrong, status, says):
    assert call(lib, **wrong) == status
    assert says in lib.ttpa_last_error(), lib.ttpa_last_error()


@pytest.mark.parametrize("call, wrong", [(_rope, dict(tokens=1 << 25)), (_update, dict(users=1 << 25)), (_fill, dict(s=1 << 30, bs=16, w=1 << 26))])
def test_more_than_one_launch_takes_is_refused(lib, call, wrong):
    assert call(lib, **wrong) == -1
    assert b"too many" in lib.ttpa_last_error(), lib.ttpa_last_error()


def test_nothing_to_do_is_no_error(lib):
    assert _rope(lib, tokens=0) == 0 and _fill(lib, users=0) == 0 and _fill(lib, s=0) == 0 and _update(lib, users=0) == 0


def test_workspace_sizes(lib):
    size = lib.ttpa_paged_fp8_sparse_decode_workspace_bytes
    assert 0 < size(2, 8, 2, 128, 8, 4) < size(200, 8, 2, 128, 8, 4) <= size(2000, 8, 2, 128, 8, 4)
    assert size(2000, 8, 2, 128, 8, 4) == size(1024, 8, 2, 128, 8, 4)  # passes of at most 2048 (user, KV head) pairs
    assert size(0, 8, 2, 128, 8, 4) == 0 and size(2, 7, 2, 128, 8, 4) == 0
    chunk = lib.ttpa_chunked_fp8_attention_workspace_bytes
    assert chunk(1, 8, 2, 32, 128, 64, 16, 0) > chunk(1, 8, 2, 32, 128, 64, 16, 100) > 2 * 2 * 64 * 128 * 2 * 2
    assert chunk(0, 8, 2, 32, 128, 64, 16, 0) == 0


def test_the_reference_codec_is_e4m3():
    """The tests' own rounding against torch's conversion on the CPU, for every bfloat16 number in range."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    assert torch.equal(R.nearest_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    s = R.scale_for(torch.tensor([[[448.0]], [[449.0]], [[0.0]], [[float("inf")]], [[1.0]], [[3e38]]]).double())
    assert s.tolist() == [1.0, 2.0, 2.0**-110, 2.0**-110, 2.0**-8, 2.0**119]


def test_rope_table():
    from tt_xla_amd.fp8_ops import rope_table

    t = rope_table(5, 8, 100.0, "cpu", torch.float64)
    for p in range(5):
        for j in range(4):
            a = p * 100.0 ** (-2 * j / 8)
            assert abs(float(t[p, j]) - float(torch.tensor(a).double().cos())) < 1e-7
            assert abs(float(t[p, 4 + j]) - float(torch.tensor(a).double().sin())) < 1e-7
