"""nitrix_amd -- MI355X-native (gfx950) fused scaled-dot-product attention.

A drop-in for nitrix's attention path (``nitrix.nn.attention``) and its
sibling fused selective scan (``nitrix.nn.ssm``): the same call signatures,
backed by hand-written HIP kernels behind a C ABI (``include/nxattn.h``,
``libnxattn.so``).  Beyond the reference: attention over packed sequences with
grouped heads (``packed_attention``), rotary positions (``rotary_embed``) and a
paged key-value cache (``paged_attention``, ``write_pages`` and the page
operators), in the model's type or in 4 or 8 bits (``write_quantized_pages``,
``read_quantized_pages``, ``quantized_paged_attention``).
"""

from ._backend import (
    NitrixBackendError,
    NitrixBackendFallback,
    reproducible,
    reset_fallback_state,
    resolve_backend,
)
from .attention import (
    HipNotTileable,
    default_scale,
    qk_rms_norm,
    reference_scaled_dot_product_attention,
    scaled_dot_product_attention,
    scaled_dot_product_attention_hip,
)
from .packed import (
    packed_attention,
    packed_attention_hip,
    reference_packed_attention,
)
from .paged import (
    compact_pages,
    copy_pages,
    extend_sequences,
    fork_sequences,
    free_sequences,
    paged_attention,
    write_pages,
)
from .quantized import (
    quantized_paged_attention,
    read_quantized_pages,
    write_quantized_pages,
)
from .rotary import (
    packed_positions,
    reference_rotary_embed,
    rotary_embed,
    rotary_frequencies,
)
from .ssm import (
    reference_selective_scan,
    selective_scan,
    selective_scan_hip,
)

__all__ = [
    'HipNotTileable',
    'NitrixBackendError',
    'NitrixBackendFallback',
    'compact_pages',
    'copy_pages',
    'default_scale',
    'extend_sequences',
    'fork_sequences',
    'free_sequences',
    'packed_attention',
    'packed_attention_hip',
    'packed_positions',
    'paged_attention',
    'qk_rms_norm',
    'quantized_paged_attention',
    'read_quantized_pages',
    'reference_packed_attention',
    'reference_rotary_embed',
    'reference_scaled_dot_product_attention',
    'reference_selective_scan',
    'reproducible',
    'reset_fallback_state',
    'resolve_backend',
    'rotary_embed',
    'rotary_frequencies',
    'scaled_dot_product_attention',
    'scaled_dot_product_attention_hip',
    'selective_scan',
    'selective_scan_hip',
    'write_pages',
    'write_quantized_pages',
]
