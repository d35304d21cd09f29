"""MI355X-native sliding-window 2-simplicial attention (gfx950 HIP kernels behind the
Python API of lucidrains/simplicial-attention for that one path)."""
from .adamw import AdamW, adamw_step, state_8bit
from .cross_entropy import linear_cross_entropy
from .naive import naive_two_simplicial_attend, nth_order_attend, signed_determinant
from .paged import OutOfPages, PagedBatch, PagedCache, copy_pages, paged_append, paged_attn, paged_two_simplicial_attn
from .rms_norm import add_rms_norm, add_rms_norm_8bit
from .sampling import sample_tokens
from .simplicial_mha import HigherOrderAttention, TwoSimplicialMHA
from .two_simplicial_attention import (
    SlidingTwoSimplicialAttention,
    SlidingWindowTwoSimplicialMHA,
    sliding_two_simplicial_attn,
)

__all__ = [
    'naive_two_simplicial_attend',
    'nth_order_attend',
    'signed_determinant',
    'HigherOrderAttention',
    'TwoSimplicialMHA',
    'SlidingTwoSimplicialAttention',
    'SlidingWindowTwoSimplicialMHA',
    'sliding_two_simplicial_attn',
    'OutOfPages',
    'PagedBatch',
    'PagedCache',
    'copy_pages',
    'paged_append',
    'paged_attn',
    'paged_two_simplicial_attn',
    'sample_tokens',
    'linear_cross_entropy',
    'add_rms_norm',
    'add_rms_norm_8bit',
    'AdamW',
    'adamw_step',
    'state_8bit',
]
