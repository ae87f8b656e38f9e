"""Block swap on the host: caches of every element type move bit for bit, an 8-bit layer with its scales and bounds."""

import pytest
import torch

import __graft_entry__  # noqa: F401  (puts the package on sys.path)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _noise(g, *shape, dtype):
    size = torch.empty((), dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=g, dtype=torch.uint8).view(dtype)


def _layer(g, nb, dtype):
    hkv, bs, d = 2, 16, 64
    kv = [_noise(g, nb, hkv, bs, d, dtype=dtype) for _ in range(2)]
    if dtype.itemsize == 1 and dtype.is_floating_point:
        kv += [_noise(g, nb, hkv, dtype=torch.float32) for _ in range(2)] + [_noise(g, nb, hkv, 2, d, dtype=torch.bfloat16)]
    return kv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.float8_e4m3fn, torch.float8_e5m2])
def test_blocks_there_and_back(dtype):
    from tt_xla_amd.kv_blocks import copy_kv_blocks

    g = torch.Generator().manual_seed(3)
    there, here = ({"a": _layer(g, nb, dtype), "b": tuple(_layer(g, nb, dtype)), "c": _layer(g, nb, dtype)[0]} for nb in (12, 6))
    lists = lambda caches: [t for v in caches.values() for t in (v if isinstance(v, (list, tuple)) else [v])]  # noqa: E731
    before, held = [t.clone() for t in lists(there)], [t.clone() for t in lists(here)]
    copy_kv_blocks(there, here, [3, 7, 1], [0, 5, 2], "d2h")
    for was, old, now in zip(before, held, lists(here)):
        assert torch.equal(_bytes(now)[[0, 5, 2]], _bytes(was)[[3, 7, 1]]) and torch.equal(_bytes(now)[[1, 3, 4]], _bytes(old)[[1, 3, 4]])
    copy_kv_blocks(here, there, [0, 5, 2], [9, 10, 11], "h2d")
    for was, now in zip(before, lists(there)):
        assert torch.equal(_bytes(now)[[9, 10, 11]], _bytes(was)[[3, 7, 1]]) and torch.equal(_bytes(now)[:9], _bytes(was)[:9])


@pytest.mark.parametrize("src, dst", [(torch.float8_e4m3fn, torch.uint8), (torch.float8_e4m3fn, torch.bfloat16), (torch.uint8, torch.float8_e4m3fn)])
def test_caches_of_different_types_are_refused(src, dst):
    """Bytes of one type are not elements of another."""
    from tt_xla_amd.kv_blocks import copy_kv_blocks

    g = torch.Generator().manual_seed(4)
    a, b = {"a": _noise(g, 4, 2, 16, 64, dtype=src)}, {"a": _noise(g, 4, 2, 16, 64, dtype=dst)}
    with pytest.raises((RuntimeError, ValueError)):
        copy_kv_blocks(a, b, [1], [2], "d2h")


def test_a_side_without_scales_is_refused():
    from tt_xla_amd.kv_blocks import copy_kv_blocks

    g = torch.Generator().manual_seed(6)
    layer = _layer(g, 4, torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="tensors"):
        copy_kv_blocks({"a": layer}, {"a": [t.clone() for t in layer[:2]]}, [1], [2], "d2h")


@pytest.mark.gpu
def test_an_8_bit_layer_to_the_host_and_back():
    from tt_xla_amd.kv_blocks import copy_kv_blocks

    g = torch.Generator().manual_seed(5)
    dev = {"a": [t.cuda() for t in _layer(g, 12, torch.float8_e4m3fn)]}
    host = {"a": [torch.zeros(6, *t.shape[1:], dtype=torch.uint8).view(t.dtype) if t.dtype.itemsize == 1 else torch.zeros(6, *t.shape[1:], dtype=t.dtype)
                  for t in dev["a"]]}
    before = [t.clone() for t in dev["a"]]
    copy_kv_blocks(dev, host, [3, 7, 1], [0, 5, 2], "d2h")
    copy_kv_blocks(host, dev, [0, 5, 2], [9, 10, 11], "h2d")
    for was, now in zip(before, dev["a"]):
        assert torch.equal(_bytes(now)[[9, 10, 11]], _bytes(was)[[3, 7, 1]]) and torch.equal(_bytes(now)[:9], _bytes(was)[:9])
