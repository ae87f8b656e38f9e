"""The 8-bit cache's fill with a length per row on the host: its schema, what tracing sees, and what its C entry point refuses before any launch."""

import pytest
import torch

import __graft_entry__ as entry


@pytest.fixture(scope="module")
def lib():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401
    from tt_xla_amd import _native

    return _native.lib()


def test_schema(lib):
    assert str(torch.ops.tt.paged_fill_fp8_cache_.lens._schema) == (
        "tt::paged_fill_fp8_cache_.lens(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales, Tensor k_fill, Tensor v_fill, Tensor page_table, "
        "Tensor? batch_idx, Tensor(e!)? key_bounds, *, Tensor lens) -> ()")


def test_tracing_and_cpu_tensors(lib):
    from torch._subclasses.fake_tensor import FakeTensorMode

    def operands():
        e = torch.zeros(4, 2, 32, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
        k = torch.zeros(1, 2, 9, 64, dtype=torch.bfloat16)
        return (e, e.clone(), torch.ones(4, 2), torch.ones(4, 2), k, k, torch.zeros(1, 2, dtype=torch.int32), None, None), torch.zeros(1, dtype=torch.int32)

    with FakeTensorMode():
        args, lens = operands()
        assert torch.ops.tt.paged_fill_fp8_cache_.lens(*args, lens=lens) is None
    args, lens = operands()
    with pytest.raises(NotImplementedError):
        torch.ops.tt.paged_fill_fp8_cache_.lens(*args, lens=lens)


# arguments that are in order, by name; pointers are aligned numbers that nothing follows (every call below is refused first)
def _fill(lib, k=16, users=2, bidx=16, lens=16, s=100, bs=64, d=128, w=4, token_stride=512):
    return lib.ttpa_paged_fill_fp8_cache_lens(16, 16, 16, 16, None, k, 51200, 128, token_stride, 16, 51200, 128, 512, 16, 4, bidx, 0, lens, 0, users, 2, 2, s, bs,
                                              d, w, 8, None)


@pytest.mark.parametrize("wrong, status, says", [
    (dict(k=None), -1, b"null"), (dict(k=8), -1, b"aligned"), (dict(bidx=None), -1, b"batch_idx"), (dict(s=257), -1, b"does not fit"), (dict(bs=40), -2, b"block_size"),
    (dict(users=-1), -1, b"dimension"), (dict(users=40000), -1, b"too many"), (dict(token_stride=500), -1, b"strides")])
def test_refused_before_any_launch(lib, wrong, status, says):
    assert _fill(lib, **wrong) == status
    assert says in lib.ttpa_last_error(), lib.ttpa_last_error()


def test_calls_of_nothing(lib):
    assert _fill(lib, users=0) == 0 and _fill(lib, s=0) == 0 and _fill(lib, s=0, lens=None) == 0
