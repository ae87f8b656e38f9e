"""Rotation by several axes with every number of head groups that a wavefront takes (``tt::qk_norm_rope_axes``): two at each head size, and four, of four and of eight groups.  Formula and tolerance are
those of ``test_gpu_rope_axes.py``."""

import pytest
import torch

import __graft_entry__ as entry
import test_gpu_rope_axes as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _pkg():
    entry.ensure_built()
    import tt_xla_amd  # noqa: F401


@pytest.mark.parametrize("hq, hk, d, rotary, tokens", [(16, 16, 128, 128, 2051), (48, 16, 128, 64, 1025), (8, 8, 256, 256, 2051), (40, 24, 64, 32, 2049), (16, 16, 64, 64, 4099),
                                                       (4, 4, 256, 128, 4099), (8, 8, 128, 128, 4097)])
@pytest.mark.parametrize("kind", ["sections", "alternating"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_groups_of_heads(hq, hk, d, rotary, tokens, kind, interleaved):
    g = torch.Generator().manual_seed(tokens + hq)
    both = torch.randn(tokens, hq + hk + 1, d, generator=g).to(torch.bfloat16)
    q, k = both[:, :hq], both[:, hq : hq + hk]
    table, pairs = T._table(300, rotary), T._pair_axes(kind, rotary // 2, 3)
    pos = torch.randint(-2, 305, (3, tokens), generator=g)
    kw = 1 + 0.2 * torch.randn(d, generator=g)
    on = both.cuda()
    got = torch.ops.tt.qk_norm_rope_axes(on[:, :hq], on[:, hq : hq + hk], table.cuda(), pos.cuda(), pairs.cuda(), None, kw.cuda(), 1e-6, interleaved)
    T._check(got[0], q, None, table, pos, pairs, 1e-6, interleaved)
    T._check(got[1], k, kw, table, pos, pairs, 1e-6, interleaved)
    torch.ops.tt.qk_norm_rope_axes_(on[:, :hq], on[:, hq : hq + hk], table.cuda(), pos.cuda(), pairs.cuda(), None, kw.cuda(), 1e-6, interleaved)
    assert torch.equal(on[:, :hq], got[0]) and torch.equal(on[:, hq : hq + hk], got[1]) and torch.equal(on[:, -1].cpu(), both[:, -1])
