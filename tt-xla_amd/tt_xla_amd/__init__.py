"""MI355X-native paged KV-cache write and paged attention behind tt-xla's operator
and attention-backend interface.

Importing the package registers the ``torch.ops.tt.*`` operators for HIP devices
(``custom_ops``, around the 8-bit cache ``fp8_ops``, for models with images, sound or video ``media_ops``); ``attention`` and ``attention_mla`` hold the vLLM-facing backend classes and ``metadata``
the host-side construction of their per-pass page tables and positions.  Every operator
runs a hand-written gfx950 kernel from ``lib/libttpa.so``; there is no other
implementation to fall back to, and a missing library is an error.
"""

from . import _native  # noqa: F401
from . import custom_ops  # noqa: F401
from . import fp8_ops  # noqa: F401
from . import media_ops  # noqa: F401
from .attention import TTAttentionBackend, TTAttentionBackendImpl, TTMetadata  # noqa: F401
from .attention_mla import TTMLAAttentionBackend, TTMLAAttentionBackendImpl  # noqa: F401
from .kv_blocks import CachePages, copy_cache_blocks, copy_kv_blocks  # noqa: F401
from .metadata import CrossMetadataBuilder, PagedMetadataBuilder  # noqa: F401

__all__ = ["TTAttentionBackend", "TTAttentionBackendImpl", "TTMLAAttentionBackend",
           "TTMLAAttentionBackendImpl", "TTMetadata", "PagedMetadataBuilder", "CrossMetadataBuilder", "CachePages", "copy_cache_blocks",
           "copy_kv_blocks", "custom_ops", "fp8_ops", "media_ops"]
