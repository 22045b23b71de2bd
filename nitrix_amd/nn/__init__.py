"""``nitrix.nn`` import path for the attention and selective-scan entry
points (``src/nitrix/nn/__init__.py:30-44`` of the reference)."""

from ..attention import (
    reference_scaled_dot_product_attention,
    scaled_dot_product_attention,
)
from ..packed import packed_attention, reference_packed_attention
from ..paged import (
    compact_pages,
    copy_pages,
    extend_sequences,
    fork_sequences,
    free_sequences,
    paged_attention,
    write_pages,
)
from ..quantized import (
    quantized_paged_attention,
    read_quantized_pages,
    write_quantized_pages,
)
from ..rotary import packed_positions, rotary_embed, rotary_frequencies
from ..ssm import reference_selective_scan, selective_scan

__all__ = [
    'compact_pages',
    'copy_pages',
    'extend_sequences',
    'fork_sequences',
    'free_sequences',
    'packed_attention',
    'packed_positions',
    'paged_attention',
    'quantized_paged_attention',
    'read_quantized_pages',
    'reference_packed_attention',
    'reference_scaled_dot_product_attention',
    'reference_selective_scan',
    'rotary_embed',
    'rotary_frequencies',
    'scaled_dot_product_attention',
    'selective_scan',
    'write_pages',
    'write_quantized_pages',
]
