"""``torch.ops.tt.*`` operators around the 8-bit cache, and helpers for its tensors.

The operators are registered by the native host module (``csrc/operators.cpp``), which loads with this package; here are
their fake implementations for tracing and what a program needs around them:

``fp8_empty_cache``, ``fp8_empty_key_bounds``
    the tensors of a layer's cache: K or V elements (``torch.float8_e4m3fn``) with a power-of-two scale for each block of tokens and
    head, and the bounds of every block's keys that the sparse decode reads.
``fp8_unpack_cache``
    the bfloat16 values that a cache stands for.
``rope_table``
    cosines and sines of positions, as the rotating operators take them.

Like the other operators these run on HIP tensors only and have no backward pass.  A cache holds e4m3 elements
[num_blocks, kv_heads, block_size, head_size]; an element stands for itself times the scale [num_blocks, kv_heads] of its block and head.
"""

from __future__ import annotations

import os
from typing import Optional

import torch

from . import _native

def fp8_empty_cache(num_blocks: int, num_kv_heads: int, block_size: int, head_size: int, device):
    """(elements, scales) of a cache of zeros."""
    elements = torch.zeros((num_blocks, num_kv_heads, block_size, head_size), dtype=torch.uint8, device=device)
    return elements.view(torch.float8_e4m3fn), torch.zeros((num_blocks, num_kv_heads), dtype=torch.float32, device=device)


def fp8_empty_key_bounds(num_blocks: int, num_kv_heads: int, head_size: int, device):
    """The least and the largest key of every block and head, feature by feature; written by the cache writers."""
    return torch.zeros((num_blocks, num_kv_heads, 2, head_size), dtype=torch.bfloat16, device=device)


def fp8_unpack_cache(elements: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values of a cache as bfloat16 (exact: an element's four significant bits times a power of two)."""
    return (elements.to(torch.float32) * scales[:, :, None, None]).to(torch.bfloat16)


def rope_table(positions: int, rotary: int, base: float = 10000.0, device=None, dtype=torch.float32) -> torch.Tensor:
    """[positions, rotary]: row p holds cos(p f_j), j < rotary / 2, then sin(p f_j), with f_j = base^(-2 j / rotary).  Angles
    are formed in 64 bits: at position 10^5 a float's own spacing is a hundredth of a turn's last digit that a float result keeps."""
    frequencies = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * frequencies
    return torch.cat([angles.cos(), angles.sin()], dim=1).to(dtype)


# --------------------------------------------------------------------------- #
# what tracing sees
# --------------------------------------------------------------------------- #
def _fresh(t: torch.Tensor) -> torch.Tensor:
    return t.new_empty(t.shape)


_registered = False


def register() -> None:
    """Loads the native module that defines the operators; once.  (Importing the package does, if it has been built.)"""
    global _registered
    if _registered:
        return
    _native.host()
    _registered = True

    @torch.library.register_fake("tt::qk_norm_rope")
    def _(query, key, cos_sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
        return _fresh(query), _fresh(key)

    @torch.library.register_fake("tt::qk_norm_rope_")
    def _(query, key, cos_sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
        return None

    @torch.library.register_fake("tt::qk_norm_rope_update_fp8_")
    def _(query, key, value, cos_sin, positions, k_cache, v_cache, k_scales, v_scales, page_table, q_weight=None,
          k_weight=None, key_bounds=None, eps=1e-6, interleaved=False):
        return _fresh(query)

    @torch.library.register_fake("tt::paged_update_fp8_cache_")
    def _(k_cache, v_cache, k_scales, v_scales, k_fill, v_fill, update_indices, page_table, key_bounds=None):
        return None

    @torch.library.register_fake("tt::paged_fill_fp8_cache_")
    def _(k_cache, v_cache, k_scales, v_scales, k_fill, v_fill, page_table, batch_idx=None, key_bounds=None):
        return None

    @torch.library.register_fake("tt::paged_fill_fp8_cache_.lens")
    def _(k_cache, v_cache, k_scales, v_scales, k_fill, v_fill, page_table, batch_idx, key_bounds, *, lens):
        return None

    @torch.library.register_fake("tt::paged_fp8_attention_decode")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, cur_pos_tensor, attention_sink=None, scale=None,
          sliding_window_size=None):
        return _fresh(query)

    @torch.library.register_fake("tt::paged_fp8_attention_decode_out")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, cur_pos_tensor, out, attention_sink=None, scale=None,
          sliding_window_size=None):
        return None

    def _columns(query, k_cache, page_table, kept_blocks):
        return page_table.new_empty((query.shape[1], k_cache.shape[1], kept_blocks), dtype=torch.int32)

    @torch.library.register_fake("tt::paged_fp8_sparse_attention_decode")
    def _(query, k_cache, v_cache, k_scales, v_scales, key_bounds, page_table, cur_pos_tensor, kept_blocks, scale=None):
        return _fresh(query), _columns(query, k_cache, page_table, kept_blocks)

    @torch.library.register_fake("tt::paged_fp8_sparse_attention_decode_out")
    def _(query, k_cache, v_cache, k_scales, v_scales, key_bounds, page_table, cur_pos_tensor, out, kept_blocks, scale=None):
        return _columns(query, k_cache, page_table, kept_blocks)

    @torch.library.register_fake("tt::chunked_fp8_attention")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, chunk_start_idx_tensor, scale=None, most_keys=0):
        return torch.empty_like(query)

    @torch.library.register_fake("tt::chunked_fp8_attention_out")
    def _(query, k_cache, v_cache, k_scales, v_scales, page_table, chunk_start_idx_tensor, out, scale=None, most_keys=0):
        return None


if os.path.exists(_native.HOST_PATH):  # (without it there are no such operators: calling one is an error)
    register()
