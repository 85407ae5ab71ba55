"""A paged cache in 8 bits, and the attention of one new token a sequence over it: paged_attention at half its memory (no counterpart in the reference).

k_pages, v_pages [P,page,Hk,N] torch.float8_e4m3fn: page a power of two, N a multiple of 16 up to 128, the innermost dimension dense, the other
strides multiples of 16.  A value is its code times the scale of its page and head, k_scales, v_scales [P,Hk] fp32."""

from ._call import ops


def WRITE(k, v, k_pages, v_pages, k_scales, v_scales, slots):
    """Puts k, v [n,Hk,N] (bf16 or fp16; strides multiples of 8) into the cache: token i at slots[i] (int32 [n]; as page_tables.EXTEND makes them), that
    is page slots[i] // page, row slots[i] % page; one outside the cache is left out.  New tokens of a page stand beside each other in the list (with none that
    is left out between them, either: two runs of a page would race for its scale), no page comes twice in it and no slot.

    The scale of a page and head is the least power of two, from 2^-100 on, that holds its finite values up to 448.  Where a page holds tokens before the first
    new one, its scale does not fall, and where it grows they are rounded once more.  What is not finite becomes NaN.  No gradients."""
    ops().cache8_write(k, v, k_pages, v_pages, k_scales, v_scales, slots)


def RUN_CUDA(q, k_pages, v_pages, k_scales, v_scales, table, lens, slopes=None, cap=0.0, scale=None):
    """y [B,H,N] of q [B,H,N] (bf16 or fp16, dense), the query of the last of each sequence's lens[b] tokens (int32 [B]), which are all in the cache; table,
    scores and what is not seen as for paged_attention.RUN_CUDA.  Scales lie between 2^-100 and 2^120, as WRITE makes them.  No gradients."""
    return ops().paged_attention8(q, k_pages, v_pages, k_scales, v_scales, table, lens, slopes, cap, scale)
