"""Page tables and slots of a batch of requests, made on the GPU from their lengths: the tables that paged_attention and paged_attention8 read, and the
slots that paged_attention8.WRITE writes to (no counterpart in the reference)."""

from ._call import ops


def EXTEND(lens, more, table, pool, taken, page, n):
    """(slots [n], starts [B+1], held [B], taken [1]), all int32, for requests that hold lens [B] tokens and get more [B] (either below 0 counts as none).

    table [B,M] names each row's pages; new ones, pool[taken[0]] (pool [F], taken [1]) and those behind it, for row 0, then row 1, ..., are written to it.
    slots names the place of every new token, row after row: page number times `page` (a power of two) plus the place in the page, -1 behind the last
    token.  starts: where each row's begin in that list, and its end.  held: the lengths afterwards; a row takes what M pages hold.  The result's taken is how many
    pages of the pool are given out then.

    What runs out is found on the GPU, where no error can be raised: a result above F says that the pool had too few pages; those are -1 in the table, and
    their tokens have slot -1, which paged_attention8.WRITE leaves out.  Tokens beyond n have no slot: starts[B] above n tells."""
    return ops().tables_extend(lens, more, table, pool, taken, page, n)
