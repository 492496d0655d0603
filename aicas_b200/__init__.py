"""aicas_b200: sm_100a attention backend for the Qwen3-VL-2B inference hot path.

Public surface = the reference package ``triton_qwen3vl``'s ``__all__``
(triton_qwen3vl/__init__.py:1-16 in the reference project) plus the operators
it leaves to Hugging Face or lacks: :func:`rope_kv_append`,
:func:`gqa_decode_partial` and :func:`merge_partials`, and the decode-side
products of its native decode path (:func:`decode_linear`).  A paged cache
(:func:`paged_rope_kv_append`, :func:`paged_gqa_decode_attention`) holds more
requests in the same memory, and 4-bit weights (:func:`decode_linear_int4`) make
a decode step read a quarter of the bytes.  A cache of 4-bit rows
(:func:`paged_rope_kv_append_int4`, :func:`paged_gqa_decode_attention_int4`) does the
same for long contexts, and eviction by attention weight
(:func:`paged_attention_weights`, :func:`paged_kv_evict`) bounds their length.
"""
from . import _native
from .backends import TEXT_BACKEND_KEY, VISION_BACKEND_KEY, text_triton_attention, vision_triton_attention
from .eviction import paged_attention_weights, paged_kv_evict
from .int4 import Int4Weight, decode_linear_int4, quantize_int4
from .ops import (
    decode_linear,
    gqa_decode_attention,
    gqa_decode_partial,
    gqa_flash_attention,
    merge_partials,
    rope_kv_append,
    varlen_flash_attention,
    vision_rope,
)
from .paged import PagedKVCache, paged_gqa_decode_attention, paged_rope_kv_append
from .paged_int4 import (
    Int4Pages,
    int4_pages,
    paged_gqa_decode_attention_int4,
    paged_kv_read_int4,
    paged_rope_kv_append_int4,
    quantize_kv_int4,
)
from .patch import install_qwen3vl_triton_attention


def __getattr__(name: str):
    """``TRITON_AVAILABLE`` / ``NATIVE_AVAILABLE``: in the reference the first
    says whether Triton imported (dense_flash_attention.py:7-15); here both say
    whether the native library loads.  They are computed on first use, so that
    importing the package (for its seeded workloads, say) maps no library."""
    if name in ("TRITON_AVAILABLE", "NATIVE_AVAILABLE"):
        return _native.available()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")

__all__ = [
    "Int4Pages",
    "Int4Weight",
    "NATIVE_AVAILABLE",
    "PagedKVCache",
    "TEXT_BACKEND_KEY",
    "TRITON_AVAILABLE",
    "VISION_BACKEND_KEY",
    "decode_linear",
    "decode_linear_int4",
    "gqa_decode_attention",
    "gqa_decode_partial",
    "gqa_flash_attention",
    "install_qwen3vl_triton_attention",
    "int4_pages",
    "merge_partials",
    "paged_attention_weights",
    "paged_gqa_decode_attention",
    "paged_gqa_decode_attention_int4",
    "paged_kv_evict",
    "paged_kv_read_int4",
    "paged_rope_kv_append",
    "paged_rope_kv_append_int4",
    "quantize_int4",
    "quantize_kv_int4",
    "rope_kv_append",
    "text_triton_attention",
    "varlen_flash_attention",
    "vision_rope",
    "vision_triton_attention",
]
