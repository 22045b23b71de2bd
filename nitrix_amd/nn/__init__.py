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
from ..ssm import reference_selective_scan, selective_scan

__all__ = [
    'compact_pages',
    'copy_pages',
    'extend_sequences',
    'fork_sequences',
    'free_sequences',
    'packed_attention',
    'paged_attention',
    'reference_packed_attention',
    'reference_scaled_dot_product_attention',
    'reference_selective_scan',
    'scaled_dot_product_attention',
    'selective_scan',
    'write_pages',
]
