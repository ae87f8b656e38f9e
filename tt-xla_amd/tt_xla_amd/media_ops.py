"""``torch.ops.tt.*`` operators of models that read images, sound or video beside a text, and helpers for their operands.

The operators are registered by the native host module (``csrc/operators.cpp``); here are their fake implementations for tracing:

``tt::qk_norm_rope_axes``, ``tt::qk_norm_rope_axes_``
    norm and rotation as ``tt::qk_norm_rope``, every pair of features by the position on its axis (time, height, width).
``tt::paged_cross_attention``, ``tt::paged_cross_attention_out``, ``tt::paged_fp8_cross_attention``, ``tt::paged_fp8_cross_attention_out``
    attention to an encoder's states in a paged cache of bfloat16 values or of one byte per element, a length per user and no causal limit.
``tt::copy_cache_blocks_``, ``tt::keep_cache_tokens_``
    copies of whole blocks, and compaction of sequences, in the caches of all layers at once (``kv_blocks.CachePages`` plans them).

``rope_pair_axes``
    the axis of every pair of features, as the rotating operators take it.

Like the other operators these run on HIP tensors only and have no backward pass.
"""

from __future__ import annotations

import os
from typing import Sequence

import torch

from . import _native, fp8_ops


def rope_pair_axes(sections: Sequence[int], alternating: bool = False, device=None) -> torch.Tensor:
    """[rotary / 2] int32: the axis of every pair.  ``sections[a]`` pairs belong to axis a; one axis behind the other, or
    ``alternating``: the axes take turns along the pairs, each until its section is used up, and the first one takes what is left."""
    if not sections or min(sections) < 0 or sum(sections) <= 0:
        raise ValueError(f"sections must hold the number of pairs of every axis, got {list(sections)}")
    if not alternating:
        return torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(list(sections))).to(device=device, dtype=torch.int32)
    pairs = torch.zeros(sum(sections), dtype=torch.int32)
    for axis, n in enumerate(sections):
        if axis and axis + (n - 1) * len(sections) >= len(pairs):
            raise ValueError(f"axis {axis} has no {n} turns in {len(pairs)} pairs of {len(sections)} axes")
        if axis:
            pairs[axis : axis + n * len(sections) : len(sections)] = axis
    return pairs.to(device)


# --------------------------------------------------------------------------- #
# what tracing sees
# --------------------------------------------------------------------------- #
_registered = False


def register() -> None:
    """Loads the native module that defines the operators; once.  (Importing the package does, if it has been built.)"""
    global _registered
    if _registered:
        return
    fp8_ops.register()
    _registered = True

    @torch.library.register_fake("tt::qk_norm_rope_axes")
    def _(query, key, cos_sin, positions, pair_axes, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
        return query.new_empty(query.shape), key.new_empty(key.shape)

    @torch.library.register_fake("tt::qk_norm_rope_axes_")
    def _(query, key, cos_sin, positions, pair_axes, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
        return None

    @torch.library.register_fake("tt::paged_cross_attention")
    def _(query, key, value, page_table, encoder_lens, scale=None, most_keys=0):
        return torch.empty_like(query)

    @torch.library.register_fake("tt::paged_cross_attention_out")
    def _(query, key, value, page_table, encoder_lens, out, scale=None, most_keys=0):
        return None

    @torch.library.register_fake("tt::paged_fp8_cross_attention")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, encoder_lens, scale=None, most_keys=0):
        return torch.empty_like(query)

    @torch.library.register_fake("tt::paged_fp8_cross_attention_out")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, encoder_lens, out, scale=None, most_keys=0):
        return None

    @torch.library.register_fake("tt::copy_cache_blocks_")
    def _(caches, source_blocks, target_blocks):
        return None

    @torch.library.register_fake("tt::keep_cache_tokens_")
    def _(caches, page_table, kept, kept_lens, first=None):
        return None


if os.path.exists(_native.HOST_PATH):  # (without it there are no such operators: calling one is an error)
    register()
