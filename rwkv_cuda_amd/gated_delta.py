"""Gated delta rule, bf16 or fp16 (no counterpart in the reference; its place is beside rwkv7, whose state it shares and whose update it gates by head):

    S_t = e^{g_t} S_{t-1};  u_t = beta_t (v_t - S_t^T k_t);  S_t += k_t u_t^T;  y_t = scale S_t^T q_t

q, k [B,T,Hk,N], v [B,T,H,N] with H a multiple of Hk (head h reads head h Hk / H) and N a multiple of 8 up to 128; the innermost dimension
dense, the other strides multiples of 8 (views of one projection).  g (a log decay) and beta [B,T,H].  Keys are taken as they are: with lengths above
1 and beta above 1 the state may grow without bounds.  Below -104 a log decay is a decay of 0, as exp gives it in fp32; above 0 it lets the state
grow, and e to the sum of 64 of them in a row must be an fp32 number.

`doc` [B,T] int32 names the document of each token of a packed or padded batch, as for gated_recurrence.RUN_CUDA: where it changes, a
document starts from a state of zero; a negative one is padding, whose y is 0 and which leaves the state as it is, whatever stands there.  Not even an
infinity or NaN passes from one document to another, in either direction, nor a decay of nothing; within its document it may reach up to 63 tokens before it
(behind it, in the gradients).  Rows with such values are done again token by token where they have documents, padding or decays of nothing: some 2 us a token."""

import torch

from ._call import ops


class GATED_DELTA(torch.autograd.Function):
    """apply(q, k, v, g, beta, s0, doc, scale) -> (y [B,T,H,N], sT [B,H,N,N] fp32, key by value); s0 [B,H,N,N] fp32 or None (zeros); gradients of q, k,
    v, g, beta and s0."""

    @staticmethod
    def apply(q, k, v, g, beta, s0=None, doc=None, scale=None):
        return ops().gated_delta(q, k, v, g, beta, s0, doc, scale)


def RUN_CUDA(q, k, v, g, beta, s0=None, doc=None, scale=None):
    """scale None: 1 / sqrt(N)."""
    return GATED_DELTA.apply(q, k, v, g, beta, s0, doc, scale)


def STEP(q, k, v, g, beta, s, out=None, scale=None):
    """One token a sequence, for serving: q, k [B,Hk,N], v [B,H,N], g, beta [B,H], s [B,H,N,N] fp32.  Returns y [B,H,N]; the new state goes to
    `out`, or replaces s where that is None; `out` is another memory than the other tensors and (unless it is s itself) s.  No gradients."""
    return ops().gated_delta_step(q, k, v, g, beta, s, s if out is None else out, scale)
