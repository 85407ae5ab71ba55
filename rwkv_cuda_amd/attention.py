"""Attention, bf16 or fp16, for the attention layers between recurrent ones (no counterpart in the reference):

    s = scale q.k,  s = cap tanh(s / cap),  s -= slopes[h] |i - j|,  y = softmax(s) v over the visible keys

q [B,Tq,H,N], k, v [B,Tk,Hk,N] with H a multiple of Hk (head h reads key head h Hk / H) and N a multiple of 8 up to 128; the innermost
dimension dense, the other strides multiples of 8 (views of one projection).  The queries are the last Tq of the Tk positions.

Visible are all keys, or, with `causal`, those up to the query's own position and those before prefix[b] (int32 [B]; below 0 is as 0).  `doc` [B,Tk] int32
names the document of each token: a query sees its own document's keys only; a negative one is padding, which sees nothing (y = 0) and
is not seen, whatever stands there.  (A NaN or an infinity in a real token may reach every row of its batch element and head, as in any
product with weights of 0.)  Gradients of q, k and v."""

import torch

from ._call import ops


class ATTENTION(torch.autograd.Function):
    """apply(q, k, v, doc, prefix, slopes, cap, scale, causal) -> y [B,Tq,H,N]"""

    @staticmethod
    def apply(q, k, v, doc=None, prefix=None, slopes=None, cap=0.0, scale=None, causal=True):
        return ops().attention(q, k, v, doc, prefix, slopes, cap, scale, causal)


def RUN_CUDA(q, k, v, doc=None, prefix=None, slopes=None, cap=0.0, scale=None, causal=True):
    """cap 0: scores are not capped, else from 2^-20 to 4096; scale None: 1 / sqrt(N), else above 0 up to 2^60 and, with slopes, from 2^-60."""
    return ATTENTION.apply(q, k, v, doc, prefix, slopes, cap, scale, causal)
