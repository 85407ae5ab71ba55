"""Gated linear recurrence, channel by channel, bf16, fp16 or fp32 (no counterpart in the reference; its place is beside the WKV ops):

    h_t = a_t h_{t-1} + u_t,  y_t = h_t        a = sigmoid(w) or exp(w),  u = (1 - a) x (tied) or x

`doc` [B,T] int32 names the document of each token of a packed or padded batch, as for attention.RUN_CUDA: where it changes, a
document starts from a state of zero; a negative one is padding, whose y is 0 and which the state passes by.

Gates are multiplied over runs of up to T tokens in fp32.  With log gates above 0 such a product may exceed it, and is then an infinity to every
state but one of exactly zero."""

import torch

from ._call import ops

GATES = ("sigmoid", "log")


def _gate(gate):
    if gate not in GATES:
        raise ValueError(f"gate must be one of {GATES}, got {gate!r}")
    return GATES.index(gate)


class GATED_RECURRENCE(torch.autograd.Function):
    """apply(w, x, h0, doc, gate, tied) -> (y [B,T,C], hT [B,C] fp32); w, x [B,T,C] of one dtype, any strides with dense channels;
    h0 [B,C] fp32 or None (zeros); gradients of w, x and h0."""

    @staticmethod
    def apply(w, x, h0=None, doc=None, gate="sigmoid", tied=True):
        return ops().gated_recurrence(w, x, h0, doc, _gate(gate), tied)


def RUN_CUDA(w, x, h0=None, doc=None, gate="sigmoid", tied=True):
    return GATED_RECURRENCE.apply(w, x, h0, doc, gate, tied)


def STEP(w, x, h, out=None, gate="sigmoid", tied=True):
    """One token a sequence, for serving: w, x [B,C], h [B,C] fp32.  Returns y [B,C]; the new state goes to `out`, or replaces h where
    that is None; `out` is another memory than w, x and (unless it is h itself) h.  No gradients."""
    return ops().gated_recurrence_step(w, x, h, h if out is None else out, _gate(gate), tied)
