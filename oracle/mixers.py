"""The gated recurrence, attention and paged attention in 64 bits, token by token and pair by pair, with error bounds.

No counterpart in the reference: each function restates the definition of the package's docstrings (gated_recurrence.py,
attention.py, paged_attention.py).  tests/test_oracle_mixers.py pins the gradients against differences and autograd.

Every function returns {name: (value, bound)}: `bound` is how far a kernel may be off that computes in 32 bits and rounds once at the end
(attention: also the softmax's weights, and the gradients of the scores, once each, before they are multiplied).  U32 = 2^-24 is half a step of
fp32 relative to the value, UNIT[dtype] that of the output's type, TINY[dtype] half of its smallest step.
"""
import math

import torch

U32 = 2.0 ** -24
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
# fp32 roundings a step of the recurrence can add, relative to its terms: exponential, sum and quotient of the gate 2 + 1 + 2, the product and
# the sum of the step 2, the composition of steps 2; with a spare factor below 2 for the hardware's exponential (2 steps instead of half a one)
ROUNDINGS = 16
# Below fp32's least normal number, 2^-126, nothing is relative to the value any more: a product of decays that falls below it may be lost whole,
# together with the state or gradient (under 2^6 in magnitude) that it multiplies, in each of up to 2^20 steps.
LEAST = 2.0 ** -100


def _gates(w, gate):
    return (torch.sigmoid(w), torch.sigmoid(-w)) if gate == "sigmoid" else (torch.exp(w), -torch.expm1(w))


def gated_recurrence(w, x, h0=None, doc=None, gate="sigmoid", tied=True, dy=None, dhT=None):
    """y, hT and, with dy or dhT, dw, dx, dh0.  Bounds: an error e_t of the state obeys e_t = a_t e_{t-1} + ROUNDINGS U32 (a_t |h|_{t-1} + |u_t|),
    |h| being the state of the magnitudes; one of its gradient the same backwards."""
    dt = w.dtype
    w, x = w.detach().double(), x.detach().double()
    B, T, C = w.shape
    dev = w.device
    real = torch.ones(B, T, dtype=torch.bool, device=dev) if doc is None else doc >= 0
    first = torch.zeros_like(real)
    if doc is not None:
        first[:, 1:] = real[:, 1:] & (doc[:, 1:] != doc[:, :-1])
    a, rest = _gates(w, gate)
    u = rest * x if tied else x
    zero = torch.zeros(B, C, dtype=torch.float64, device=dev)
    h = zero if h0 is None else h0.detach().double()
    m, e = h.abs(), zero
    keep = {n: torch.zeros(B, T, C, dtype=torch.float64, device=dev) for n in ("y", "ey", "hp", "mp", "ep")}
    c = ROUNDINGS * U32
    for t in range(T):
        r, f = real[:, t, None], first[:, t, None]
        hp, mp, ep = (torch.where(f, zero, z) for z in (h, m, e))
        hn = a[:, t] * hp + u[:, t]
        mn = a[:, t] * mp + u[:, t].abs()
        en = a[:, t] * ep + c * (a[:, t] * mp + u[:, t].abs())
        h, m, e = (torch.where(r, n, o) for n, o in ((hn, h), (mn, m), (en, e)))
        keep["y"][:, t], keep["ey"][:, t] = torch.where(r, h, zero), torch.where(r, e, zero)
        keep["hp"][:, t], keep["mp"][:, t], keep["ep"][:, t] = hp, mp, ep
    out = {"y": (keep["y"], UNIT[dt] * keep["y"].abs() + TINY[dt] + LEAST + keep["ey"]), "hT": (h, e + U32 * h.abs() + LEAST)}
    if dy is None and dhT is None:
        return out
    g = torch.zeros(B, T, C, dtype=torch.float64, device=dev) if dy is None else dy.double()
    d = zero if dhT is None else dhT.double()
    md, ed = d.abs(), zero
    grads = {n: torch.zeros(B, T, C, dtype=torch.float64, device=dev) for n in ("dw", "ew", "dx", "ex")}
    slope = a * rest if gate == "sigmoid" else a
    for t in range(T - 1, -1, -1):
        r, f = real[:, t, None], first[:, t, None]
        dn = d + g[:, t]
        mn = md + g[:, t].abs()
        en = ed + c * mn
        hp, mp, ep = keep["hp"][:, t], keep["mp"][:, t], keep["ep"][:, t]
        z = hp - x[:, t] if tied else hp
        mz = mp + x[:, t].abs() if tied else mp
        k = rest[:, t].abs() if tied else 1.0
        grads["dw"][:, t] = torch.where(r, dn * z * slope[:, t], zero)
        grads["ew"][:, t] = torch.where(r, slope[:, t].abs() * (en * mz + mn * (ep + c * mz)), zero)
        grads["dx"][:, t] = torch.where(r, dn * (rest[:, t] if tied else 1.0), zero)
        grads["ex"][:, t] = torch.where(r, (en + c * mn) * k, zero)
        cut = torch.where(f, zero, a[:, t])
        d, md, ed = (torch.where(r, cut * n, o) for n, o in ((dn, d), (mn, md), (en + c * mn, ed)))
    out["dw"] = (grads["dw"], UNIT[dt] * grads["dw"].abs() + TINY[dt] + LEAST + grads["ew"])
    out["dx"] = (grads["dx"], UNIT[dt] * grads["dx"].abs() + TINY[dt] + LEAST + grads["ex"])
    if h0 is not None:
        out["dh0"] = (d, ed + U32 * d.abs() + LEAST)
    return out


def visible(Tq, Tk, doc=None, prefix=None, causal=True, device="cpu"):
    """[Tq,Tk] for one row of the batch: doc [Tk] or None, prefix an int or None."""
    at = torch.arange(Tk - Tq, Tk, device=device)[:, None]
    j = torch.arange(Tk, device=device)[None, :]
    on = torch.ones(Tq, Tk, dtype=torch.bool, device=device)
    if causal:
        on = j <= at
        if prefix is not None:
            on = on | (j < prefix)
    if doc is not None:
        on = on & (doc[None, :] == doc[Tk - Tq:, None]) & (doc[None, :] >= 0)
    return on


def _least_operands(v, dy, doc, dt):
    """Half of the smallest step of the scores' gradients and of the weights as operands of one batch element, fp16.  The former are taken times a power of two that brings
    the largest |dy| |v| + |dy.y| (lengths of rows) of queries and keys that are no padding to 2^14 .. 2^15; |dy.y| is at most |dy| times the largest |v|, to the roundings of y.  The
    latter are taken times 2^8."""
    if dt != torch.float16:
        return TINY[dt], TINY[dt]

    def longest(z, doc):
        n = z.detach().double().norm(dim=-1)
        n = n if doc is None else n[doc >= 0]
        n = n[torch.isfinite(n)]
        return float(n.max()) if n.numel() else 0.0
    most = 2.02 * longest(dy, None if doc is None else doc[-dy.shape[0]:]) * longest(v, doc)
    return TINY[dt] * most * 2.0 ** -14, TINY[dt] * 2.0 ** -8


def _head(q, k, v, on, dist, slope, cap, scale, do, dt, least=(0.0, 0.0)):
    """One head: y, its bound, and with do the four pieces of the gradients with theirs.  `least`: what the gradients of the scores and the weights may be off by as
    operands of the gradients' products, beside their relative rounding."""
    u, tiny, N = UNIT[dt], TINY[dt], q.shape[1]
    lost = 2.0 ** -126                                         # a weight below fp32's least normal number may be lost whole
    raw = (q @ k.T) * scale
    s = cap * torch.tanh(raw / cap) if cap else raw
    # sums of N products and the scale; the cap's tanh and quotient, to 8 roundings of the cap; bias, maximum, and base change of the exponential
    es = (N + 4) * U32 * scale * (q.abs() @ k.abs().T) + (8 * U32 * cap if cap else 0.0) + 4 * U32 * s.abs()
    if slope is not None:
        s = s - slope * dist
        es = es + 4 * U32 * slope * dist
    s = torch.where(on, s, torch.full_like(s, -math.inf))
    some = on.any(1, keepdim=True)
    top = torch.where(some, s.amax(1, keepdim=True), torch.zeros_like(s[:, :1]))
    p = torch.exp(s - top)
    # the maximum is subtracted in fp32, and the exponential is off by 4 steps
    es = torch.where(on, es, torch.zeros_like(es)) + 4 * U32 * (1 + top.abs())
    total = p.sum(1, keepdim=True)
    p = torch.where(some, p / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(p))
    worst = es.amax(1, keepdim=True)
    rel = 2 * (es + worst) + 16 * U32                          # of a weight: its own error and the sum's
    y = p @ v
    n = on.sum(1, keepdim=True).clamp(min=1).sqrt()
    ey = u * y.abs() + tiny + u * (p @ v.abs()) + (p * rel) @ v.abs() + (tiny + lost) * (on.double() @ v.abs()) + 8 * U32 * n * (p @ v.abs())
    if do is None:
        return y, ey
    dp = do @ v.T
    delta = (do * y).sum(1, keepdim=True)
    edp = (N + 4) * U32 * (do.abs() @ v.abs().T)
    # delta comes from y as the forward wrote it in two parts, off by u^2 of the weights' rounding and by u of what those are off
    edelta = (do.abs() * ((N + 4) * U32 * y.abs() + ey - u * y.abs() + u * u * y.abs() + 2 * tiny)).sum(1, keepdim=True)
    t1 = 1 - torch.tanh(raw / cap) ** 2 if cap else torch.ones_like(raw)
    ds = p * (dp - delta) * t1
    seen = on.double()
    # 1 - t^2: off by twice the tanh's error
    eds = p * t1 * (edp + edelta) + ds.abs() * rel + (p * (dp - delta).abs() * 24 * U32 if cap else 0.0) + lost * seen * (1 + (dp - delta).abs())

    def back(w, ew, on, z, least):                             # w @ z with w rounded to the type before
        return w @ z, (u * w.abs() + ew + least * on) @ z.abs()
    dq, eq = back(ds, eds, seen, k, least[0])
    dk, ek = back(ds.T, eds.T, seen.T, q, least[0])
    dv, ev = back(p.T, (p * rel + lost * seen).T, seen.T, do, least[1])
    more = 8 * U32 * math.sqrt(max(on.shape))                  # the fp32 sums of the three products
    eq, ek, ev = eq + more * (ds.abs() @ k.abs()), ek + more * (ds.T.abs() @ q.abs()), ev + more * (p.T @ do.abs())
    return y, ey, (scale * dq, scale * eq), (scale * dk, scale * ek), (dv, ev)


def attention(q, k, v, doc=None, prefix=None, slopes=None, cap=0.0, scale=None, causal=True, dy=None):
    """y and, with dy, dq, dk, dv."""
    dt = q.dtype
    B, Tq, H, N = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(N) if scale is None else scale
    u, tiny = UNIT[dt], TINY[dt]
    Q, K, V = (z.detach().double() for z in (q, k, v))
    new = lambda like: [torch.zeros(like.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
    y, gq, gk, gv = new(q), new(q), new(k), new(k)
    dist = (torch.arange(Tk - Tq, Tk, device=q.device)[:, None] - torch.arange(Tk, device=q.device)[None, :]).abs().double()
    for b in range(B):
        on = visible(Tq, Tk, None if doc is None else doc[b], None if prefix is None else int(prefix[b]), causal, q.device)
        least = (0.0, 0.0) if dy is None else _least_operands(v[b], dy[b], None if doc is None else doc[b], dt)
        for h in range(H):
            g = h * Hk // H
            r = _head(Q[b, :, h], K[b, :, g], V[b, :, g], on, dist, None if slopes is None else float(slopes[h]), cap, scale,
                      None if dy is None else dy[b, :, h].double(), dt, least)
            y[0][b, :, h], y[1][b, :, h] = r[0], r[1]
            if dy is None:
                continue
            gq[0][b, :, h], gq[1][b, :, h] = r[2]
            for z, part in ((gk, r[3]), (gv, r[4])):
                z[0][b, :, g] += part[0]
                z[1][b, :, g] += part[1]
    out = {"y": (y[0], y[1])}
    if dy is not None:
        for n, z in (("dq", gq), ("dk", gk), ("dv", gv)):
            out[n] = (z[0], z[1] + u * z[0].abs() + tiny)
    return out


def paged_attention(q, k_pages, v_pages, table, lens, slopes=None, cap=0.0, scale=None):
    """y: each sequence's tokens gathered from its pages (those of pages out of range left out), then one row of attention."""
    dt = q.dtype
    B, H, N = q.shape
    P, page, Hk, _ = k_pages.shape
    scale = 1 / math.sqrt(N) if scale is None else scale
    y = [torch.zeros(B, H, N, dtype=torch.float64, device=q.device) for _ in range(2)]
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        at = torch.arange(min(n, table.shape[1] * page), device=q.device)
        rows = table[b].long()[at // page]
        fine = (rows >= 0) & (rows < P)
        at, rows = at[fine], rows[fine]
        if not len(at):
            continue
        dist = (n - 1 - at)[None, :].double()
        on = torch.ones(1, len(at), dtype=torch.bool, device=q.device)
        for h in range(H):
            g = h * Hk // H
            k, v = k_pages[rows, at % page, g].double(), v_pages[rows, at % page, g].double()
            y[0][b, h], y[1][b, h] = (z[0] for z in _head(q[b, h][None].double(), k, v, on, dist, None if slopes is None else float(slopes[h]), cap, scale, None, dt))
    return {"y": (y[0], y[1])}
