"""Attention of one new token a sequence over a cache in pages, bf16 or fp16: what attention.RUN_CUDA is in serving (no counterpart in
the reference)."""

from ._call import ops


def RUN_CUDA(q, k_pages, v_pages, table, lens, k=None, v=None, slopes=None, cap=0.0, scale=None):
    """y [B,H,N] of q [B,H,N], dense, the query of the last of each sequence's lens[b] tokens (int32 [B]).

    k_pages, v_pages [P,page,Hk,N]: page a power of two, N a multiple of 8 up to 128, the innermost dimension dense, the other strides
    multiples of 8.  Token t of sequence b is row t % page of page table[b, t // page] (int32 [B,M]).  With k and v [B,Hk,N], dense, the new
    token's key and value are written to the cache, at lens[b] - 1, and count from there; a page that is written must belong to one
    sequence, in one place.

    A sequence with lens[b] <= 0 has y = 0.  Tokens beyond the table's pages, and tokens of pages that are not in 0 .. P-1, are left out
    (they are found on the GPU, where no error can be raised).  No gradients."""
    return ops().paged_attention(q, k_pages, v_pages, table, lens, k, v, slopes, cap, scale)
