"""Where the device plans a cross attention's parts (host side, seen in the scratch that a call asks for): its estimate counts steps in floats, which hold whole numbers up to 2^24, and
the room for parts, twice the CUs' workgroups and one per user and KV head, is right for exact counts alone.  600 users and heads of 2^24 + 1 steps each, cut by 2^24, would be two parts each: more
than there is room for."""

import pytest

import __graft_entry__ as entry


@pytest.fixture(scope="module")
def lib():
    entry.ensure_built()
    from tt_xla_amd import _native

    return _native.lib()


@pytest.mark.parametrize("d, step", [(128, 64), (256, 32)])  # keys of a step where workgroups share their tiles
@pytest.mark.parametrize("steps, planned", [((1 << 24) - 128, True), (1 << 24, False), ((1 << 24) + 128, False)])
def test_lengths_that_floats_do_not_count_are_not_planned(lib, d, step, steps, planned):
    slot = 64 * (d + 2) * 4  # a part of a block of rows: accumulators, maxima and sums; the plan stands in front of them
    for most_keys, width in ((0, steps * step // 4096), (steps * step, 1 << 19)):
        bytes_ = lib.ttpa_paged_cross_attention_workspace_bytes(3, 64, 1, 1, d, 4096, width, most_keys)
        assert bytes_ > 0 and (bytes_ % slot != 0) == planned


def test_a_float_below_the_longest_cut_would_not_fit():
    """The arithmetic of the bound: parts of 600 equal users and heads, 256 CUs, one block of rows."""
    import struct

    as_float = lambda x: struct.unpack("f", struct.pack("f", x))[0]  # noqa: E731
    segments, room = 600, 2 * 256 + 1 + 600
    for steps, fits in (((1 << 24) - 1, True), ((1 << 24) + 1, False)):
        share = int(as_float(steps))
        assert (segments * -(-steps // share) <= room) == fits
