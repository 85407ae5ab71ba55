"""What the speed of the sequence mixers beside the WKV family is measured on: the gated linear recurrence, attention with capped
scores, distance bias, documents and prefixes, and the attention of one new token over a paged cache.

A case is a dict of plain values.  `run` computes the operators in plain torch operations, or, with `own`, through the package.
All inputs live in GPU memory and are drawn there from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # serving: the next token of 32 conversations in one recurrent layer; nothing but the call's latency
        dict(name="recurrence_token", op="recurrence", dtype="bf16", B=32, T=1, C=2048, gate="sigmoid", tied=True, state=True, docs=0, pad=0, fused=False, train=False),
        # fine-tuning on one packed row: documents of odd lengths, padding behind them, gate and input views of one projection
        dict(name="recurrence_docs", op="recurrence", dtype="fp16", B=1, T=3001, C=2048, gate="sigmoid", tied=False, state=True, docs=5, pad=37, fused=True, train=True),
        # prefill of one long text in fp32, decays given as logarithms
        dict(name="recurrence_prefill", op="recurrence", dtype="fp32", B=1, T=65536, C=1024, gate="log", tied=True, state=True, docs=0, pad=0, fused=False, train=False),
        # a training layer at the batch, length and width of the package's other layers
        dict(name="recurrence_layer", op="recurrence", dtype="bf16", B=8, T=4096, C=4096, gate="sigmoid", tied=True, state=False, docs=0, pad=0, fused=False, train=True),
        # one GPU's micro-batch of a small model, scores biased by distance
        dict(name="attention_small", op="attention", dtype="bf16", B=4, Tq=512, Tk=512, H=12, Hk=12, N=64, causal=True, cap=0.0, bias=True, docs=0, pad=0, prefix=False, fused=False, train=True),
        # fine-tuning on one packed row: documents of odd lengths, padding, capped scores, shared key heads, views of one projection
        dict(name="attention_docs", op="attention", dtype="fp16", B=1, Tq=3001, Tk=3001, H=32, Hk=8, N=128, causal=True, cap=30.0, bias=False, docs=5, pad=37, prefix=False, fused=True, train=True),
        # a training layer with heads of 64 at the batch and length of the package's other layers
        dict(name="attention_layer", op="attention", dtype="bf16", B=8, Tq=4096, Tk=4096, H=32, Hk=32, N=64, causal=True, cap=0.0, bias=True, docs=0, pad=0, prefix=False, fused=False, train=True),
        # a training layer on long sequences whose first part is seen from everywhere, shared key heads, capped scores
        dict(name="attention_prefix", op="attention", dtype="bf16", B=2, Tq=8192, Tk=8192, H=32, Hk=8, N=128, causal=True, cap=50.0, bias=False, docs=0, pad=0, prefix=True, fused=False, train=True),
        # prefill in pieces: the last 512 tokens of a long prompt against all of its keys
        dict(name="attention_piece", op="attention", dtype="bf16", B=1, Tq=512, Tk=16384, H=32, Hk=8, N=128, causal=True, cap=0.0, bias=False, docs=0, pad=0, prefix=False, fused=False, train=False),
        # serving one conversation of ordinary length: latency
        dict(name="paged_one", op="paged", dtype="bf16", B=1, longest=1000, H=32, Hk=8, N=128, page=16, cap=0.0, bias=False, append=False),
        # serving many conversations of all lengths, the new token's key and value written on the way, a key head per head
        dict(name="paged_many", op="paged", dtype="bf16", B=64, longest=4096, H=32, Hk=32, N=64, page=16, cap=0.0, bias=True, append=True),
        # serving a few very long texts
        dict(name="paged_long", op="paged", dtype="fp16", B=4, longest=131072, H=64, Hk=8, N=128, page=64, cap=30.0, bias=False, append=False),
    ]


# a drawn case costs no more than the largest listed one of its operator
MAX_ELEMS = 8 * 4096 * 4096
MAX_PAIRS = 2 * 32 * 128 * 8192 * 4100
MAX_CACHE = 4 * 131072 * 8 * 128


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["recurrence", "attention", "paged"])
    while True:
        if op == "recurrence":
            T = _log_int(rng, 1, 65536)
            docs = rng.choice([0, 0, 3, 9]) if T >= 64 else 0
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), B=_log_int(rng, 1, 64), T=T, C=_log_int(rng, 32, 4096), gate=rng.choice(["sigmoid", "log"]),
                        tied=rng.random() < 0.5, state=rng.random() < 0.5, docs=docs, pad=rng.choice([0, 11]) if docs else 0, fused=rng.random() < 0.3,
                        train=rng.random() < 0.7)
            if case["B"] * T * case["C"] * (2 if case["dtype"] == "fp32" else 1) <= MAX_ELEMS:
                return case
        elif op == "attention":
            Tk = _log_int(rng, 1, 16384)
            Tq = Tk if rng.random() < 0.7 else _log_int(rng, 1, Tk)
            Hk = _log_int(rng, 1, 16)
            H = Hk * rng.choice([1, 1, 2, 4, 8])
            docs = rng.choice([0, 0, 3, 9]) if Tk >= 64 else 0
            causal = rng.random() < 0.8
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=_log_int(rng, 1, 16), Tq=Tq, Tk=Tk, H=H, Hk=Hk, N=rng.choice([64, 64, 128, 128, 32, 80, 96]), causal=causal,
                        cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.random() < 0.4, docs=docs, pad=rng.choice([0, 11]) if docs else 0,
                        prefix=causal and rng.random() < 0.3, fused=Tq == Tk and rng.random() < 0.3, train=rng.random() < 0.6)
            if case["B"] * H * case["N"] * Tq * Tk <= MAX_PAIRS and H <= 64:
                return case
        else:
            Hk = _log_int(rng, 1, 32)
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=_log_int(rng, 1, 128), longest=_log_int(rng, 1, 131072), H=Hk * rng.choice([1, 2, 4, 8, 16]), Hk=Hk,
                        N=rng.choice([64, 64, 128, 128, 32, 80, 96]), page=rng.choice([16, 32, 64, 256]), cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.3,
                        append=rng.random() < 0.3)
            cache = case["B"] * case["longest"] * Hk * case["N"]
            if cache <= (MAX_CACHE // 16 if case["append"] else MAX_CACHE) and case["H"] <= 128:
                return case


# ------------------------------------------------------------------------------------------------ inputs
def _doc_ids(T, docs, pad):
    """Documents of uneven lengths over the first T - pad tokens, -1 behind them."""
    if not docs:
        return None
    n = T - pad
    cuts = sorted({(n * (i * i + 3 * i + 1)) // (docs * docs + 3 * docs + 1) for i in range(1, docs)})
    ids = torch.zeros(T, dtype=torch.int32)
    for c in cuts:
        ids[c:] += 1
    ids[n:] = -1
    return ids


def _lengths(case):
    """From the longest down to a few tokens, in no order."""
    B, n = case["B"], case["longest"]
    return [max(1, n - (n * ((7 * b) % B)) // (B + 1)) for b in range(B)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    dt, B = DTYPES[case["dtype"]], case["B"]
    state = dict(case=case)
    if case["op"] == "recurrence":
        T, C = case["T"], case["C"]
        # gates around 0.88, or time constants around 20 tokens with a spread of a factor of 3
        w = normal(B, T, C) + 2.0 if case["gate"] == "sigmoid" else -torch.exp(normal(B, T, C) - 3.0)
        x = normal(B, T, C)
        if case["fused"]:
            both = torch.cat([w, x], 2).to(dt)
            w, x = both[..., :C], both[..., C:]
        state.update(w=w.to(dt), x=x.to(dt), h0=normal(B, C) if case["state"] else None)
        doc = _doc_ids(T, case["docs"], case["pad"])
        state["doc"] = None if doc is None else doc.to(DEV).expand(B, T).contiguous()
        if case["train"]:
            state["dy"] = normal(B, T, C).to(dt)
            state["dhT"] = normal(B, C) if case["state"] else None
            state["leaves"] = [state[n].requires_grad_(True) for n in ("w", "x", "h0") if state[n] is not None]
        if T == 1:
            state["h1"] = torch.empty(B, C, device=DEV)
        return state
    H, Hk, N = case["H"], case["Hk"], case["N"]
    # one slope a head, from 1/2 downwards: the far past is left to the heads with small ones
    state["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H) if case["bias"] else None
    if case["op"] == "attention":
        Tq, Tk = case["Tq"], case["Tk"]
        if case["fused"]:
            x = normal(B, Tq, (H + 2 * Hk) * N).to(dt)
            q, k, v = (z.unflatten(2, (-1, N)) for z in x.split([H * N, Hk * N, Hk * N], 2))
        else:
            q, k, v = normal(B, Tq, H, N).to(dt), normal(B, Tk, Hk, N).to(dt), normal(B, Tk, Hk, N).to(dt)
        state.update(q=q, k=k, v=v)
        doc = _doc_ids(Tk, case["docs"], case["pad"])
        state["doc"] = None if doc is None else doc.to(DEV).expand(B, Tk).contiguous()
        state["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device=DEV) if case["prefix"] else None
        if case["train"]:
            state["dy"] = normal(B, Tq, H, N).to(dt)
            state["leaves"] = [z.requires_grad_(True) for z in (q, k, v)]
        return state
    lens, page = _lengths(case), case["page"]
    pages = [-(-n // page) for n in lens]
    total = sum(pages)
    state["k_pages"] = torch.empty(total, page, Hk, N, device=DEV, dtype=dt)
    state["v_pages"] = torch.empty(total, page, Hk, N, device=DEV, dtype=dt)
    for z in (state["k_pages"], state["v_pages"]):
        z.normal_(generator=g)
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    state.update(table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV), host_lens=lens, q=normal(B, H, N).to(dt))
    state["k"], state["v"] = (normal(B, Hk, N).to(dt), normal(B, Hk, N).to(dt)) if case["append"] else (None, None)
    return state


def _prefixes(case):
    return [max(1, case["Tk"] * (b + 1) // (8 * case["B"])) for b in range(case["B"])]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _recurrence_own(state):
    from rwkv_cuda_amd import gated_recurrence
    case = state["case"]
    if case["T"] == 1 and case["state"] and not case["train"] and not case["docs"]:
        y = gated_recurrence.STEP(state["w"][:, 0], state["x"][:, 0], state["h0"], out=state["h1"], gate=case["gate"], tied=case["tied"])
        return [y.unsqueeze(1), state["h1"]]
    if not case["train"]:
        with torch.no_grad():
            return list(gated_recurrence.RUN_CUDA(state["w"], state["x"], state["h0"], state["doc"], gate=case["gate"], tied=case["tied"]))
    y, hT = gated_recurrence.RUN_CUDA(state["w"], state["x"], state["h0"], state["doc"], gate=case["gate"], tied=case["tied"])
    grads = torch.autograd.grad([y, hT] if case["state"] else [y], state["leaves"], [state["dy"], state["dhT"]] if case["state"] else [state["dy"]])
    return [y.detach(), hT.detach()] + list(grads)


def _attention_own(state):
    from rwkv_cuda_amd import attention
    case = state["case"]
    how = dict(doc=state["doc"], prefix=state["prefix"], slopes=state["slopes"], cap=case["cap"], causal=case["causal"])
    if not case["train"]:
        with torch.no_grad():
            return [attention.RUN_CUDA(state["q"], state["k"], state["v"], **how)]
    y = attention.RUN_CUDA(state["q"], state["k"], state["v"], **how)
    return [y.detach()] + list(torch.autograd.grad([y], state["leaves"], [state["dy"]]))


def _paged_own(state):
    from rwkv_cuda_amd import paged_attention
    case = state["case"]
    y = paged_attention.RUN_CUDA(state["q"], state["k_pages"], state["v_pages"], state["table"], state["lens"], k=state["k"], v=state["v"], slopes=state["slopes"], cap=case["cap"])
    return [y, state["k_pages"], state["v_pages"]] if case["append"] else [y]


_own = {"recurrence": _recurrence_own, "attention": _attention_own, "paged": _paged_own}


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling: after the step with n, entry t holds the composition of the last 2n steps."""
    n, T = 1, a.shape[1]
    while n < T:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        n2 = 2 * n
        if n2 < T:
            a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n = n2
    return b


def _marks(doc):
    """Which tokens are real, and which start from nothing: real ones whose predecessor has another id."""
    real = doc >= 0
    first = torch.zeros_like(real)
    first[:, 1:] = real[:, 1:] & (doc[:, 1:] != doc[:, :-1])
    return real.unsqueeze(2), first.unsqueeze(2)


@torch.no_grad()
def _recurrence_plain(state):
    case = state["case"]
    dt, T = DTYPES[case["dtype"]], case["T"]
    w, x, h0, doc = state["w"].float(), state["x"].float(), state["h0"], state["doc"]
    if case["gate"] == "sigmoid":
        a = 1 / (1 + torch.exp(-w))
        rest = 1 / (1 + torch.exp(w))
    else:
        a, rest = torch.exp(w), -torch.expm1(w)
    u = rest * x if case["tied"] else x
    A = a
    if doc is not None:
        real, first = _marks(doc)
        A = torch.where(first, 0.0, torch.where(real, a, 1.0))
        u = torch.where(real, u, 0.0)
    b = u
    if h0 is not None:
        b = torch.cat([u[:, :1] + A[:, :1] * h0.unsqueeze(1), u[:, 1:]], 1)
    h = _scan(A, b)
    y = (h if doc is None else torch.where(real, h, 0.0)).to(dt)
    out = [y, h[:, -1].clone()]
    if not case["train"]:
        return out
    dy = state["dy"].float()
    if doc is not None:
        dy = torch.where(real, dy, 0.0)
    if state["dhT"] is not None:
        dy = torch.cat([dy[:, :-1], dy[:, -1:] + state["dhT"].unsqueeze(1)], 1)
    nxt = torch.cat([A[:, 1:], torch.zeros_like(A[:, :1])], 1)
    dh = _scan(nxt.flip(1), dy.flip(1)).flip(1)
    start = torch.zeros_like(h[:, :1]) if h0 is None else h0.unsqueeze(1)
    da = dh * torch.cat([start, h[:, :-1]], 1)
    if doc is not None:
        da = torch.where(first, 0.0, da)
    if case["tied"]:
        da = da - dh * x
    dw = da * a * rest if case["gate"] == "sigmoid" else da * a
    dx = dh * rest if case["tied"] else dh
    if doc is not None:
        dw, dx = torch.where(real, dw, 0.0), torch.where(real, dx, 0.0)
    out += [dw.to(dt), dx.to(dt)]
    if h0 is not None:
        out.append(A[:, 0] * dh[:, 0])
    return out


def _visible(state, b, Tq, Tk):
    """[Tq,Tk]: the pairs of query and key that count in row b; the queries are the last Tq positions."""
    case = state["case"]
    i = torch.arange(Tk - Tq, Tk, device=DEV).unsqueeze(1)
    j = torch.arange(Tk, device=DEV).unsqueeze(0)
    vis = j <= i if case["causal"] else torch.ones(Tq, Tk, dtype=torch.bool, device=DEV)
    if state["prefix"] is not None:
        vis = vis | (j < state["prefix"][b])
    if state["doc"] is not None:
        doc = state["doc"][b]
        vis = vis & (doc[Tk - Tq:].unsqueeze(1) == doc.unsqueeze(0)) & (doc >= 0).unsqueeze(0)
    return vis, (i - j).abs().float()


@torch.no_grad()
def _attention_plain(state):
    case = state["case"]
    dt, B, Tq, Tk, H, Hk, N, cap = DTYPES[case["dtype"]], case["B"], case["Tq"], case["Tk"], case["H"], case["Hk"], case["N"], case["cap"]
    G, scale = H // Hk, 1 / math.sqrt(N)
    q, k, v = state["q"], state["k"], state["v"]
    y = torch.empty(B, Tq, H, N, device=DEV, dtype=dt)
    if case["train"]:
        dq, dk, dv = torch.empty_like(y), torch.empty(B, Tk, Hk, N, device=DEV, dtype=dt), torch.empty(B, Tk, Hk, N, device=DEV, dtype=dt)
    # as many key heads at once as 2^28 scores allow, each with the queries of all heads that share it: [key head, head and query, key]
    step = max(1, 2 ** 28 // (G * Tq * Tk))
    for b in range(B):
        vis, dist = _visible(state, b, Tq, Tk)
        for lo in range(0, Hk, step):
            hi = min(Hk, lo + step)
            n = hi - lo
            heads = slice(lo * G, hi * G)
            rows = lambda z: z[b, :, heads].float().transpose(0, 1).reshape(n, G * Tq, N)
            back = lambda z: z.view(n * G, Tq, N).transpose(0, 1).to(dt)
            qq = rows(q)
            kk, vv = (z[b, :, lo:hi].float().transpose(0, 1).contiguous() for z in (k, v))
            s = torch.matmul(qq, kk.transpose(1, 2).contiguous()).view(n, G, Tq, Tk) * scale
            if cap:
                t = torch.tanh(s / cap)
                s = t * cap
            if state["slopes"] is not None:
                s = s - state["slopes"][heads].view(n, G, 1, 1) * dist
            s = torch.where(vis, s, -math.inf)
            top = s.amax(3, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(3, keepdim=True)
            p = (p / torch.where(total == 0, 1.0, total)).view(n, G * Tq, Tk)
            o = torch.matmul(p, vv)
            y[b, :, heads] = back(o)
            if not case["train"]:
                continue
            do = rows(state["dy"])
            dv[b, :, lo:hi] = torch.matmul(p.transpose(1, 2).contiguous(), do).transpose(0, 1).to(dt)
            ds = p * (torch.matmul(do, vv.transpose(1, 2).contiguous()) - (do * o).sum(2, keepdim=True))
            if cap:
                ds = ds * (1 - t * t).view(n, G * Tq, Tk)
            dq[b, :, heads] = back(torch.matmul(ds, kk) * scale)
            dk[b, :, lo:hi] = (torch.matmul(ds.transpose(1, 2).contiguous(), qq) * scale).transpose(0, 1).to(dt)
    return [y, dq, dk, dv] if case["train"] else [y]


@torch.no_grad()
def _paged_plain(state):
    case = state["case"]
    dt, H, Hk, N, page, cap = DTYPES[case["dtype"]], case["H"], case["Hk"], case["N"], case["page"], case["cap"]
    G, scale = H // Hk, 1 / math.sqrt(N)
    y = torch.empty(case["B"], H, N, device=DEV, dtype=dt)
    for b, n in enumerate(state["host_lens"]):
        if case["append"]:
            where = state["table"][b, (n - 1) // page].long()
            state["k_pages"][where, (n - 1) % page] = state["k"][b]
            state["v_pages"][where, (n - 1) % page] = state["v"][b]
        rows = state["table"][b, :-(-n // page)].long()
        kk = state["k_pages"][rows].flatten(0, 1)[:n].float().transpose(0, 1).contiguous()          # [Hk, n, N]
        vv = state["v_pages"][rows].flatten(0, 1)[:n].float().transpose(0, 1).contiguous()
        qq = state["q"][b].float().view(Hk, G, N)
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        if cap:
            s = torch.tanh(s / cap) * cap
        if state["slopes"] is not None:
            s = s - state["slopes"].view(Hk, G, 1) * torch.arange(n - 1, -1, -1, device=DEV).float()
        p = torch.exp(s - s.amax(2, keepdim=True))
        p = p / p.sum(2, keepdim=True)
        y[b] = torch.matmul(p, vv).view(H, N).to(dt)
    return [y, state["k_pages"], state["v_pages"]] if case["append"] else [y]


_plain = {"recurrence": _recurrence_plain, "attention": _attention_plain, "paged": _paged_plain}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Visible pairs of query and key, summed over the batch."""
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    off, n = Tk - Tq, 0
    for b in range(B):
        prefix = _prefixes(case)[b] if case["prefix"] else 0
        if case["docs"]:
            ids = _doc_ids(Tk, case["docs"], case["pad"]).tolist()
            spans, at = [], 0
            while at < Tk:
                end = at
                while end < Tk and ids[end] == ids[at]:
                    end += 1
                if ids[at] >= 0:
                    spans.append((at, end))
                at = end
        else:
            spans = [(0, Tk)]
        for lo, hi in spans:
            for i in range(max(lo, off), hi):
                n += min(hi, max(i + 1 if case["causal"] else hi, min(prefix, hi))) - lo
    return n


def work(case):
    """Each input read once, each output written once; the multiply-adds of the definition over the pairs that are visible."""
    eb = 4 if case["dtype"] == "fp32" else 2
    B = case["B"]
    if case["op"] == "recurrence":
        n = B * case["T"] * case["C"]
        states = 4 * B * case["C"] * (1 + (1 if case["state"] else 0) + (2 if case["state"] and case["train"] else 0))
        # a gate (an exponential and a division), a multiply-add and the input's weight; backward twice that and the gate's derivative
        return {"bytes": eb * n * (6 if case["train"] else 3) + states + (4 * B * case["T"] if case["docs"] else 0), "flops": n * (8 + (20 if case["train"] else 0))}
    H, Hk, N = case["H"], case["Hk"], case["N"]
    if case["op"] == "attention":
        q, k = eb * B * case["Tq"] * H * N, eb * B * case["Tk"] * Hk * N
        side = 4 * B * case["Tk"] if case["docs"] else 0
        if case["train"]:
            return {"bytes": 4 * q + 4 * k + side, "flops": 14 * N * H * _pairs(case)}
        return {"bytes": 2 * q + 2 * k + side, "flops": 4 * N * H * _pairs(case)}
    tokens = sum(_lengths(case))
    pages = 4 * sum(-(-n // case["page"]) for n in _lengths(case)) + 4 * B
    return {"bytes": 2 * eb * tokens * Hk * N + 2 * eb * B * H * N + pages + (2 * eb * B * Hk * N if case["append"] else 0), "flops": 4 * tokens * H * N}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"recurrence": _recurrence_exact, "attention": _attention_exact, "paged": _paged_exact}[case["op"]](state)


def _recurrence_exact(state):
    """Token by token, and back again."""
    case = state["case"]
    B, T, C = case["B"], case["T"], case["C"]
    if T > 8192 and case["train"]:
        return None
    w, x = state["w"].detach().double(), state["x"].detach().double()
    doc = state["doc"]
    h = torch.zeros(B, C, device=DEV, dtype=torch.float64) if state["h0"] is None else state["h0"].detach().double()
    y = torch.empty(B, T, C, device=DEV, dtype=torch.float64)
    before = torch.empty_like(y) if case["train"] else None
    alive = None
    if doc is not None:
        alive = [(doc[:, t] >= 0).unsqueeze(1).double() for t in range(T)]
        joined = [torch.ones_like(alive[0])] + [(doc[:, t] == doc[:, t - 1]).unsqueeze(1).double() for t in range(1, T)]
    gate = (lambda z: torch.sigmoid(z)) if case["gate"] == "sigmoid" else (lambda z: z.exp())
    other = (lambda z: torch.sigmoid(-z)) if case["gate"] == "sigmoid" else (lambda z: -z.expm1())
    for t in range(T):
        a = gate(w[:, t])
        u = other(w[:, t]) * x[:, t] if case["tied"] else x[:, t]
        if alive is not None:
            old = h
            h = h * joined[t]
        if before is not None:
            before[:, t] = h
        h = a * h + u
        if alive is None:
            y[:, t] = h
        else:
            y[:, t] = h * alive[t]
            h = torch.where(alive[t] > 0, h, old)
    out = [y, h]
    if not case["train"]:
        return out
    dw, dx = torch.empty_like(y), torch.empty_like(y)
    d = torch.zeros(B, C, device=DEV, dtype=torch.float64) if state["dhT"] is None else state["dhT"].double()
    for t in range(T - 1, -1, -1):
        a, o = gate(w[:, t]), other(w[:, t])
        got = d + state["dy"][:, t].double()
        if alive is not None:
            got = torch.where(alive[t] > 0, got, torch.zeros_like(got))
        slope = a * o if case["gate"] == "sigmoid" else a
        dw[:, t] = got * slope * (before[:, t] - x[:, t] if case["tied"] else before[:, t])
        dx[:, t] = got * o if case["tied"] else got
        back = got * a
        if alive is not None:
            back = torch.where(alive[t] > 0, back * joined[t], d)
        d = back
    out += [dw, dx]
    if state["h0"] is not None:
        out.append(d)
    return out


def _attention_exact(state):
    """One head at a time; the gradients by differentiating the definition."""
    case = state["case"]
    B, Tq, Tk, H, Hk, N = case["B"], case["Tq"], case["Tk"], case["H"], case["Hk"], case["N"]
    train = case["train"]
    y = torch.empty(B, Tq, H, N, device=DEV, dtype=torch.float64)
    dq = torch.empty_like(y)
    dk = torch.zeros(B, Tk, Hk, N, device=DEV, dtype=torch.float64)
    dv = torch.zeros_like(dk)
    here = torch.arange(Tq, device=DEV) + (Tk - Tq)
    keys = torch.arange(Tk, device=DEV)
    for b in range(B):
        hidden = keys[None, :] > here[:, None] if case["causal"] else torch.zeros(Tq, Tk, dtype=torch.bool, device=DEV)
        if state["prefix"] is not None:
            hidden = hidden & (keys[None, :] >= int(state["prefix"][b]))
        if state["doc"] is not None:
            mine = state["doc"][b, here]
            hidden = hidden | (mine[:, None] != state["doc"][b][None, :]) | (mine[:, None] < 0)
        empty = hidden.all(1)
        for h in range(H):
            g = h * Hk // H
            q, k, v = (z.detach().double().requires_grad_(train) for z in (state["q"][b, :, h], state["k"][b, :, g], state["v"][b, :, g]))
            with torch.set_grad_enabled(train):
                s = (q @ k.transpose(0, 1)) / math.sqrt(N)
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if state["slopes"] is not None:
                    s = s - state["slopes"][h].double() * (here[:, None] - keys[None, :]).abs().double()
                s = s.masked_fill(hidden, -math.inf).masked_fill(empty[:, None], 0.0)
                o = torch.softmax(s, 1).masked_fill(empty[:, None], 0.0) @ v
            y[b, :, h] = o.detach()
            if train:
                a, c, d = torch.autograd.grad(o, [q, k, v], state["dy"][b, :, h].double())
                dq[b, :, h] = a
                dk[b, :, g] += c
                dv[b, :, g] += d
    return [y, dq, dk, dv] if train else [y]


def _paged_exact(state):
    case = state["case"]
    H, Hk, N, page = case["H"], case["Hk"], case["N"], case["page"]
    y = torch.empty(case["B"], H, N, device=DEV, dtype=torch.float64)
    kp, vp = state["k_pages"], state["v_pages"]
    if case["append"]:
        kp, vp = kp.clone(), vp.clone()
        for b, n in enumerate(state["host_lens"]):
            spot = int(state["table"][b, (n - 1) // page])
            kp[spot, (n - 1) % page], vp[spot, (n - 1) % page] = state["k"][b], state["v"][b]
    for b, n in enumerate(state["host_lens"]):
        at = torch.arange(n, device=DEV)
        spots = state["table"][b].long()[at // page]
        for g in range(Hk):
            k, v = kp[spots, at % page, g].double(), vp[spots, at % page, g].double()
            mine = slice(g * (H // Hk), (g + 1) * (H // Hk))
            s = (state["q"][b, mine].double() @ k.transpose(0, 1)) / math.sqrt(N)
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if state["slopes"] is not None:
                s = s - state["slopes"][mine].double()[:, None] * (n - 1 - at)[None, :].double()
            y[b, mine] = torch.softmax(s, 1) @ v
    return [y, kp.double(), vp.double()] if case["append"] else [y]
