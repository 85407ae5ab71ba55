"""The gated delta rule in 64 bits, token by token, its gradients by differentiating the definition.

No counterpart in the reference: it restates the docstring of gated_delta.py.  tests/test_oracle_delta.py pins the gradients against differences."""
import math

import torch


def gated_delta(q, k, v, g, beta, s0=None, doc=None, scale=None, dy=None, dsT=None):
    """{name: value}: y, sT and, with dy or dsT, dq, dk, dv, dg, dbeta, ds0 (of a zero state where s0 is None)."""
    B, T, Hk, N = k.shape
    H = v.shape[2]
    scale = 1 / math.sqrt(N) if scale is None else scale
    grad = dy is not None or dsT is not None
    Q, K, V, G, W = leaves = [z.detach().double().requires_grad_(grad) for z in (q, k, v, g, beta)]
    S = start = (torch.zeros(B, H, N, N, dtype=torch.float64, device=v.device) if s0 is None else s0.detach().double()).requires_grad_(grad)
    head = torch.arange(H, device=v.device) * Hk // H
    real = torch.ones(B, T, dtype=torch.bool, device=v.device) if doc is None else doc >= 0
    cut = torch.zeros_like(real)
    if doc is not None:
        cut[:, 1:] = real[:, 1:] & (doc[:, 1:] != doc[:, :-1])
    cut = cut[:, :, None] | (G.detach() < -104)                  # e^g is 0 in 32 bits
    ys = []
    for t in range(T):
        on = real[:, t, None, None]
        kt, qt, vt = (torch.where(on, z, torch.zeros_like(z)) for z in (K[:, t, head], Q[:, t, head], V[:, t]))
        a = torch.where(cut[:, t], torch.zeros_like(G[:, t]), torch.where(cut[:, t], torch.zeros_like(G[:, t]), G[:, t]).exp())
        a = torch.where(real[:, t, None], a, torch.ones_like(a))
        b = torch.where(real[:, t, None], W[:, t], torch.zeros_like(W[:, t]))
        S = torch.where(cut[:, t, :, None, None] & on[..., None], torch.zeros_like(S), S * a[..., None, None])
        u = b[..., None] * (vt - (kt[..., None] * S).sum(2))
        S = S + kt[..., None] * u[:, :, None]
        ys.append(scale * (qt[..., None] * S).sum(2))
    y = torch.stack(ys, 1)
    out = dict(y=y.detach(), sT=S.detach())
    if grad:
        loss = (0 if dy is None else (y * dy.double()).sum()) + (0 if dsT is None else (S * dsT.double()).sum())
        for n, z in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), torch.autograd.grad(loss, leaves + [start], allow_unused=True)):
            out[n] = z if z is not None else torch.zeros_like(dict(zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), leaves + [start]))[n])
    return out
