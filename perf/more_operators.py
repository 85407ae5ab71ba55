"""What the speed of four more operators is measured on: the gated delta rule (whole sequences in training and prefill, and its single-token step),
a paged cache in 8 bits (writing it, and the attention of one new token a sequence over it), and the page tables and slots of a batch of requests.

A case is a dict of plain values.  `run` computes the operators in plain torch operations, or, with `own`, through the package.
All inputs live in GPU memory and are drawn there from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn


def listed():
    return [
        # serving: the next token of 32 conversations in one recurrent layer; the states are read and written
        dict(name="delta_token", op="step", dtype="bf16", B=32, H=32, Hk=16, N=128),
        # one GPU's micro-batch of a small model
        dict(name="delta_small", op="delta", dtype="bf16", B=4, T=512, H=12, Hk=12, N=64, state=True, docs=0, pad=0, fused=False, train=True),
        # fine-tuning on one packed row: documents of odd lengths, padding, shared key heads, views of one projection
        dict(name="delta_docs", op="delta", dtype="fp16", B=1, T=3001, H=32, Hk=16, N=128, state=False, docs=5, pad=37, fused=True, train=True),
        # a training layer at the batch, length and width of the package's other layers
        dict(name="delta_layer", op="delta", dtype="bf16", B=8, T=4096, H=32, Hk=32, N=64, state=False, docs=0, pad=0, fused=False, train=True),
        # prefill of one long text that goes on from a state
        dict(name="delta_prefill", op="delta", dtype="bf16", B=1, T=32768, H=32, Hk=16, N=128, state=True, docs=0, pad=0, fused=False, train=False),
        # serving: the next token of 64 conversations goes into the cache; latency
        dict(name="cache_append", op="write", dtype="bf16", B=64, longest=1000, tokens=1, Hk=8, N=128, page=16),
        # prefill: prompts of all lengths go into the cache behind what is there
        dict(name="cache_prefill", op="write", dtype="bf16", B=16, longest=500, tokens=4096, Hk=8, N=128, page=64),
        # serving one conversation of ordinary length: latency
        dict(name="cache8_one", op="paged8", dtype="bf16", B=1, longest=1000, H=32, Hk=8, N=128, page=16, cap=0.0, bias=False),
        # serving many conversations of all lengths, a key head per head, scores biased by distance
        dict(name="cache8_many", op="paged8", dtype="bf16", B=64, longest=4096, H=32, Hk=32, N=64, page=16, cap=0.0, bias=True),
        # serving a few very long texts, capped scores
        dict(name="cache8_long", op="paged8", dtype="fp16", B=4, longest=131072, H=64, Hk=8, N=128, page=64, cap=30.0, bias=False),
        # serving: a token more for each of 256 requests
        dict(name="tables_step", op="tables", B=256, longest=4000, tokens=1, M=512, page=16),
        # prompts of 1024 requests enter at once
        dict(name="tables_prompts", op="tables", B=1024, longest=300, tokens=700, M=128, page=16),
    ]


# a drawn case costs no more than the largest listed one of its operator
MAX_DELTA = 8 * 4096 * 32 * 64
MAX_STATE = 32 * 32 * 128 * 128
MAX_WRITE = 16 * 4096 * 8 * 128
MAX_CACHE = 4 * 131072 * 8 * 128
MAX_TOKENS = 1024 * 700


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "delta", "delta", "delta", "write", "paged8", "paged8", "tables"])
    while True:
        Hk = _log_int(rng, 1, 32)
        N = rng.choice([64, 64, 128, 128, 32, 80, 96])
        if op in ("step", "delta"):
            H = Hk * rng.choice([1, 1, 2, 4])
            B = _log_int(rng, 1, 64)
            if op == "step":
                case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=B, H=H, Hk=Hk, N=N)
                if B * H * N * N <= MAX_STATE and H <= 64:
                    return case
                continue
            T = _log_int(rng, 1, 32768)
            docs = rng.choice([0, 0, 3, 9]) if T >= 64 else 0
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=B, T=T, H=H, Hk=Hk, N=N, state=rng.random() < 0.5, docs=docs, pad=rng.choice([0, 11]) if docs else 0,
                        fused=rng.random() < 0.3, train=rng.random() < 0.7)
            if B * T * H * N <= MAX_DELTA and H <= 64:
                return case
        elif op == "write":
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=_log_int(rng, 1, 128), longest=_log_int(rng, 1, 4096), tokens=rng.choice([1, _log_int(rng, 1, 8192)]), Hk=Hk, N=N,
                        page=rng.choice([16, 32, 64, 256]))
            if case["B"] * case["tokens"] * Hk * N <= MAX_WRITE and case["B"] * (case["longest"] + case["tokens"]) * Hk * N <= MAX_CACHE:
                return case
        elif op == "paged8":
            case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=_log_int(rng, 1, 128), longest=_log_int(rng, 1, 131072), H=Hk * rng.choice([1, 2, 4, 8, 16]), Hk=Hk, N=N,
                        page=rng.choice([16, 32, 64, 256]), cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.3)
            if case["B"] * case["longest"] * Hk * N <= MAX_CACHE and case["H"] <= 128:
                return case
        else:
            page, tokens, longest = rng.choice([16, 32, 64, 256]), rng.choice([1, _log_int(rng, 1, 4096)]), _log_int(rng, 1, 4096)
            case = dict(op=op, B=_log_int(rng, 1, 2048), longest=longest, tokens=tokens, M=-(-(longest + tokens) // page) + rng.choice([0, 17, 100]), page=page)
            if case["B"] * tokens <= MAX_TOKENS and case["B"] * case["M"] <= 1 << 20:
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


def _spread(most, B):
    """From `most` down to a few, in no order."""
    return [max(1, most - (most * ((7 * b) % B)) // (B + 1)) for b in range(B)]


def _row_tokens(case):
    """Tokens that are there, and tokens that come, of each row of a batch of requests."""
    B = case["B"]
    held = [n - 1 for n in _spread(case["longest"], B)]
    return held, _spread(case["tokens"], B)[::-1]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"step": _prepare_delta, "delta": _prepare_delta, "write": _prepare_write, "paged8": _prepare_paged8, "tables": _prepare_tables}[case["op"]](case, g)


def _prepare_delta(case, g):
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    dt, B, T, H, Hk, N = DTYPES[case["dtype"]], case["B"], case.get("T", 1), case["H"], case["Hk"], case["N"]
    step = case["op"] == "step"
    unit = lambda z: z / z.square().sum(-1, keepdim=True).sqrt()
    # queries and keys of length 1, the keys of a head around a common direction
    q, k, v = unit(normal(B, T, Hk, N)), unit(normal(B, T, Hk, N) + 0.7 * normal(1, 1, Hk, N)), normal(B, T, H, N)
    if case.get("fused"):
        q, k, v = (z.unflatten(2, (-1, N)) for z in torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], 2).to(dt).split([Hk * N, Hk * N, H * N], 2))
    # time constants around 30 tokens, from 1 to some hundreds
    gate, beta = -torch.exp(1.2 * normal(B, T, H) - 3.5), 1 / (1 + torch.exp(-normal(B, T, H)))
    state = dict(case=case, q=q.to(dt), k=k.to(dt), v=v.to(dt), g=gate.to(dt), beta=beta.to(dt), s0=normal(B, H, N, N) * 0.3 if step or case["state"] else None)
    if step:
        for n in ("q", "k", "v", "g", "beta"):
            state[n] = state[n][:, 0]
        state["s1"] = torch.empty_like(state["s0"])
        return state
    doc = _doc_ids(T, case["docs"], case["pad"])
    state["doc"] = None if doc is None else doc.to(DEV).expand(B, T).contiguous()
    if case["train"]:
        state["dy"] = normal(B, T, H, N).to(dt)
        state["dsT"] = normal(B, H, N, N) * 0.3 if case["state"] else None
        state["leaves"] = [state[n].requires_grad_(True) for n in ("q", "k", "v", "g", "beta", "s0") if state[n] is not None]
    return state


def _pages_of(lens, page, g):
    """A table of pages in no order for rows of these lengths, and how many pages there are."""
    need = [-(-n // page) for n in lens]
    total, most = sum(need), max(need)
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    here = torch.arange(most, device=DEV).unsqueeze(0) < torch.tensor(need, device=DEV).unsqueeze(1)
    table = torch.zeros(len(lens), most, dtype=torch.int32, device=DEV)
    table[here] = order
    return table, total


def _codes(pages, page, Hk, N, g):
    """A cache of values around 1 in 8 bits: codes whose largest magnitude in a page and head lies above 224 (the scale is the least power of two
    that holds it), and scales around 2^-7."""
    x = torch.empty(pages, page, Hk, N, device=DEV, dtype=torch.float16)
    x.normal_(generator=g)
    scales = torch.exp2(torch.randint(-8, -5, (pages, Hk), generator=g, device=DEV).float())
    return (x * 90.0).clamp_(-448.0, 448.0).to(FP8), scales


def _prepare_write(case, g):
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    dt, Hk, N, page = DTYPES[case["dtype"]], case["Hk"], case["N"], case["page"]
    held, new = _row_tokens(case)
    table, P = _pages_of([a + b for a, b in zip(held, new)], page, g)
    n = sum(new)
    row = torch.repeat_interleave(torch.arange(case["B"], device=DEV), torch.tensor(new, device=DEV))
    counts = torch.tensor(new, device=DEV)
    at = torch.arange(n, device=DEV) - (counts.cumsum(0) - counts)[row] + torch.tensor(held, device=DEV)[row]
    slots = table[row, at // page].long() * page + at % page
    kp, ks = _codes(P, page, Hk, N, g)
    vp, vs = _codes(P, page, Hk, N, g)
    # a token in fifty has keys and values four times as large
    k, v = (normal(n, Hk, N) * torch.where(torch.rand(n, 1, 1, generator=g, device=DEV) < 0.02, 4.0, 1.0) for _ in range(2))
    return dict(case=case, k=k.to(dt), v=v.to(dt), k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs, slots=slots.to(torch.int32))


def _prepare_paged8(case, g):
    dt, B, H, Hk, N, page = DTYPES[case["dtype"]], case["B"], case["H"], case["Hk"], case["N"], case["page"]
    lens = _spread(case["longest"], B)
    table, P = _pages_of(lens, page, g)
    kp, ks = _codes(P, page, Hk, N, g)
    vp, vs = _codes(P, page, Hk, N, g)
    # one slope a head, from 1/2 downwards: the far past is left to the heads with small ones
    slopes = torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H) if case["bias"] else None
    return dict(case=case, q=torch.randn(B, H, N, generator=g, device=DEV).to(dt), k_pages=kp, v_pages=vp, k_scales=ks, v_scales=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                slopes=slopes)


def _prepare_tables(case, g):
    B, M, page = case["B"], case["M"], case["page"]
    held, new = _row_tokens(case)
    have = [-(-n // page) for n in held]
    need = [-(-(a + b) // page) for a, b in zip(held, new)]
    order = torch.randperm(sum(need), generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
    there = torch.arange(M, device=DEV).unsqueeze(0) < torch.tensor(have, device=DEV).unsqueeze(1)
    table[there] = order[:sum(have)]
    # the pool: all pages, those that are held first
    return dict(case=case, lens=torch.tensor(held, dtype=torch.int32, device=DEV), new=torch.tensor(new, dtype=torch.int32, device=DEV), table=table, pool=order,
                taken=torch.tensor([sum(have)], dtype=torch.int32, device=DEV), n=sum(new))


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _step_own(state):
    from rwkv_cuda_amd import gated_delta
    y = gated_delta.STEP(*(state[n] for n in ("q", "k", "v", "g", "beta")), state["s0"], out=state["s1"])
    return [y, state["s1"]]


def _delta_own(state):
    from rwkv_cuda_amd import gated_delta
    args = [state[n] for n in ("q", "k", "v", "g", "beta", "s0", "doc")]
    if not state["case"]["train"]:
        with torch.no_grad():
            return list(gated_delta.RUN_CUDA(*args))
    y, sT = gated_delta.RUN_CUDA(*args)
    grads = torch.autograd.grad([y, sT] if state["s0"] is not None else [y], state["leaves"], [state["dy"], state["dsT"]] if state["s0"] is not None else [state["dy"]])
    return [y.detach(), sT.detach()] + list(grads)


def _write_own(state):
    from rwkv_cuda_amd import paged_attention8
    cache = [state[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales")]
    paged_attention8.WRITE(state["k"], state["v"], *cache, state["slots"])
    return cache


def _paged8_own(state):
    from rwkv_cuda_amd import paged_attention8
    return [paged_attention8.RUN_CUDA(*(state[n] for n in ("q", "k_pages", "v_pages", "k_scales", "v_scales", "table", "lens")), slopes=state["slopes"], cap=state["case"]["cap"])]


def _tables_own(state):
    from rwkv_cuda_amd import page_tables
    slots, starts, held, taken = page_tables.EXTEND(*(state[n] for n in ("lens", "new", "table", "pool", "taken")), state["case"]["page"], state["n"])
    return [slots, starts, held, taken, state["table"]]


_own = {"step": _step_own, "delta": _delta_own, "write": _write_own, "paged8": _paged8_own, "tables": _tables_own}


@torch.no_grad()
def _step_plain(state):
    case = state["case"]
    dt, G, N = DTYPES[case["dtype"]], case["H"] // case["Hk"], case["N"]
    q, k = (state[n].float().repeat_interleave(G, 1) for n in ("q", "k"))
    s = state["s0"] * torch.exp(state["g"].float())[..., None, None]
    u = state["beta"].float()[..., None] * (state["v"].float() - torch.matmul(k.unsqueeze(2), s).squeeze(2))
    s = s + k.unsqueeze(3) * u.unsqueeze(2)
    return [(torch.matmul(q.unsqueeze(2), s).squeeze(2) / math.sqrt(N)).to(dt), s]


L = 64


@torch.no_grad()
def _delta_plain(state):
    """64 tokens at once: within a chunk the updates u solve a triangular system, between chunks the state goes on."""
    case = state["case"]
    dt, B, T, H, Hk, N = DTYPES[case["dtype"]], case["B"], case["T"], case["H"], case["Hk"], case["N"]
    G, C, scale = H // Hk, -(-T // L), 1 / math.sqrt(N)
    doc = state["doc"]
    real = torch.ones(B, T, dtype=torch.bool, device=DEV) if doc is None else doc >= 0
    cut = torch.zeros_like(real)
    if doc is not None:
        cut[:, 1:] = real[:, 1:] & (doc[:, 1:] != doc[:, :-1])

    def chunks(z, heads):                                       # [B,T,h,...] -> [B,H,C,L,...], nothing at padding
        z = torch.where(real.view(B, T, *[1] * (z.dim() - 2)), z.float(), 0.0)
        z = torch.cat([z, z.new_zeros(B, C * L - T, *z.shape[2:])], 1)
        z = z.view(B, C, L, *z.shape[2:]).transpose(2, 3).transpose(1, 2)
        return z.repeat_interleave(H // heads, 1) if heads != H else z.contiguous()

    q, k, v, g, beta = (chunks(state[n], Hk if n in "qk" else H) for n in ("q", "k", "v", "g", "beta"))
    cuts = torch.cat([cut, cut.new_zeros(B, C * L - T)], 1).view(B, 1, C, L)
    part = cuts.cumsum(3)
    sums = torch.where(cuts, 0.0, g).double().cumsum(3)          # log decays add up in 64 bits: their differences count
    low = torch.ones(L, L, dtype=torch.bool, device=DEV).tril()
    decay = torch.exp(torch.where(low & (part.unsqueeze(4) == part.unsqueeze(3)), (sums.unsqueeze(4) - sums.unsqueeze(3)), -math.inf).float())
    enter = torch.where(part == 0, torch.exp(sums), 0.0).float().unsqueeze(4)
    leave = torch.where(part == part[..., -1:], torch.exp(sums[..., -1:] - sums), 0.0).float().unsqueeze(4)
    whole = enter[:, :, :, -1:]
    kk, b = torch.matmul(k, k.transpose(3, 4).contiguous()), beta.unsqueeze(4)
    A = (b * decay * kk).tril(-1)
    inv = torch.eye(L, device=DEV).repeat(B, H, C, 1, 1)
    for i in range(1, L):
        inv[..., i:i + 1, :i] = -torch.matmul(A[..., i:i + 1, :i], inv[..., :i, :i])
    qk = torch.matmul(q, k.transpose(3, 4).contiguous())
    P = scale * decay * qk
    W, U = torch.matmul(inv, b * enter * k), torch.matmul(inv, b * v)
    kT = (leave * k).transpose(3, 4).contiguous()
    s = torch.zeros(B, H, N, N, device=DEV) if state["s0"] is None else state["s0"]
    S = torch.empty(B, H, C, N, N, device=DEV)
    for c in range(C):
        S[:, :, c] = s
        U[:, :, c] -= torch.matmul(W[:, :, c], s)
        s = whole[:, :, c] * s + torch.matmul(kT[:, :, c], U[:, :, c])

    def back(z, heads=H):                                       # [B,H,C,L,...] -> [B,T,h,...]
        if heads != H:
            z = z.unflatten(1, (heads, G)).sum(2)
        return z.transpose(1, 2).transpose(2, 3).reshape(B, C * L, *z.shape[1:2], *z.shape[4:])[:, :T].to(dt)

    out = [back(scale * enter * torch.matmul(q, S) + torch.matmul(P, U)), s]
    if not case["train"]:
        return out
    dy = chunks(state["dy"], H)
    ds = torch.zeros(B, H, N, N, device=DEV) if state["s0"] is None else state["dsT"]
    dS = torch.empty_like(S)                                     # of the state that leaves a chunk
    dU = torch.matmul(P.transpose(3, 4).contiguous(), dy)
    invT, Wk, kout = inv.transpose(3, 4).contiguous(), (b * enter * k).transpose(3, 4).contiguous(), leave * k
    dq_in = torch.matmul((scale * enter * q).transpose(3, 4).contiguous(), dy)
    dZ = torch.empty_like(U)
    for c in range(C - 1, -1, -1):
        dS[:, :, c] = ds
        dZ[:, :, c] = torch.matmul(invT[:, :, c], dU[:, :, c] + torch.matmul(kout[:, :, c], ds))
        ds = whole[:, :, c] * ds + dq_in[:, :, c] - torch.matmul(Wk[:, :, c], dZ[:, :, c])
    UT, ST, dST = (z.transpose(3, 4).contiguous() for z in (U, S, dS))
    dP = torch.matmul(dy, UT) * decay * scale
    dA = -torch.matmul(dZ, UT).tril(-1) * decay
    q1 = scale * enter * torch.matmul(dy, ST)
    k1 = leave * torch.matmul(U, dST)
    zS = enter * torch.matmul(dZ, ST)
    dAb = dA * b
    dq = q1 + torch.matmul(dP, k)
    dk = k1 - b * zS + torch.matmul(dP.transpose(3, 4).contiguous(), q) + torch.matmul(dAb, k) + torch.matmul(dAb.transpose(3, 4).contiguous(), k)
    dbeta = (dZ * v).sum(4) - (zS * k).sum(4) + (dA * kk).sum(4)
    # a log decay counts in all that passes its token: pairs around it, the state that enters, the state that leaves
    pairs = dP * qk + dAb * kk
    pairs = pairs.sum(4) - pairs.sum(3)
    after = (q * q1).sum(4) - b.squeeze(4) * (k * zS).sum(4) + pairs
    before = (k * k1).sum(4)
    dg = after.flip(3).cumsum(3).flip(3) + before.cumsum(3) - before + (whole * dS * S).sum((3, 4)).unsqueeze(3)
    dg = torch.where(cuts, 0.0, dg)
    hide = lambda z: torch.where(real.view(B, T, *[1] * (z.dim() - 2)), z, 0.0)
    out += [hide(back(dq, Hk)), hide(back(dk, Hk)), hide(back(b * dZ)), hide(back(dg)), hide(back(dbeta))]
    return out + [ds] if state["s0"] is not None else out


def _least_scales(top):
    """The least power of two, from 2^-100 on, by which values up to `top` fit 8 bits (up to 448)."""
    m, e = torch.frexp(top)
    e = torch.where(top > 0, torch.where(m > 0.875, e - 8, e - 9), -100).clamp(min=-100)
    return torch.ldexp(torch.ones_like(top), e)


@torch.no_grad()
def _write_plain(state):
    case = state["case"]
    page, Hk = case["page"], case["Hk"]
    slots = state["slots"].long()
    where, at = slots // page, slots % page
    P = state["k_pages"].shape[0]
    # the first of the new tokens in each page: what lies before it stays
    first = torch.full((P,), page, device=DEV).index_reduce_(0, where, at, "amin")
    some = slots.shape[0] * page < P * page
    for x, pages, scales in ((state["k"], state["k_pages"], state["k_scales"]), (state["v"], state["v_pages"], state["v_scales"])):
        top = torch.zeros(P, Hk, device=DEV).index_reduce_(0, where, x.float().abs().amax(2), "amax")
        need = _least_scales(top)
        old = scales.clone()
        scales.copy_(torch.where((first == page).unsqueeze(1), old, torch.where((first == 0).unsqueeze(1), need, torch.maximum(need, old))))
        stay = (torch.arange(page, device=DEV) < first.unsqueeze(1)) & (first < page).unsqueeze(1)
        rows = where if some else slice(None)                    # few tokens: their pages only
        raw = pages.view(torch.uint8)
        held = raw[rows].view(FP8)
        fitted = (held.float() * (old[rows] / scales[rows])[:, None, :, None]).to(FP8)
        raw[rows] = torch.where(stay[rows][:, :, None, None], fitted.view(torch.uint8), held.view(torch.uint8))
        raw[where, at] = (x.float() / scales[where].unsqueeze(2)).to(FP8).view(torch.uint8)
    return [state[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales")]


@torch.no_grad()
def _paged8_plain(state):
    case = state["case"]
    dt, B, H, Hk, N, cap = DTYPES[case["dtype"]], case["B"], case["H"], case["Hk"], case["N"], case["cap"]
    G, scale, lens, rows = H // Hk, 1 / math.sqrt(N), state["lens"].view(B, 1, 1, 1), state["table"].long()

    def values(pages, scales):                                   # [B,Hk,tokens,N]
        x = pages.view(torch.uint8)[rows].view(FP8).float() * scales[rows][:, :, None, :, None]
        return x.flatten(1, 2).transpose(1, 2).contiguous()

    kk = values(state["k_pages"], state["k_scales"])
    s = torch.matmul(state["q"].float().view(B, Hk, G, N), kk.transpose(2, 3).contiguous()) * scale
    del kk
    if cap:
        s = torch.tanh(s / cap) * cap
    at = torch.arange(s.shape[3], device=DEV)
    if state["slopes"] is not None:
        s = s - state["slopes"].view(1, Hk, G, 1) * (lens - 1 - at).float()
    s = torch.where(at < lens, s, -math.inf)
    p = torch.exp(s - s.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    return [torch.matmul(p, values(state["v_pages"], state["v_scales"])).view(B, H, N).to(dt)]


@torch.no_grad()
def _tables_plain(state):
    case = state["case"]
    B, M, page, n = case["B"], case["M"], case["page"], state["n"]
    lens, table, pool, taken = state["lens"].long(), state["table"], state["pool"], state["taken"].long()
    add = torch.minimum(state["new"].long().clamp(min=0), (M * page - lens).clamp(min=0))
    have, need = (lens + page - 1) // page, (lens + add + page - 1) // page
    more = need - have
    first = taken + more.cumsum(0) - more - have                 # page c of row b, where it is new, is number first[b] + c of the pool
    col = torch.arange(M, device=DEV).unsqueeze(0)
    at = first.unsqueeze(1) + col
    fresh = torch.where(at < pool.shape[0], pool[at.clamp(0, pool.shape[0] - 1)], -1)
    table.copy_(torch.where((col >= have.unsqueeze(1)) & (col < need.unsqueeze(1)), fresh, table))
    ends = add.cumsum(0)
    i = torch.arange(n, device=DEV)
    row = torch.searchsorted(ends, i, right=True).clamp(max=B - 1)
    t = lens[row] + i - (ends - add)[row]
    where = table[row, (t // page).clamp(max=M - 1)].long()
    slots = torch.where((i < ends[-1]) & (where >= 0), where * page + t % page, -1).to(torch.int32)
    starts = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return [slots, starts, (lens + add).to(torch.int32), (taken + more.sum()).to(torch.int32), table]


_plain = {"step": _step_plain, "delta": _delta_plain, "write": _write_plain, "paged8": _paged8_plain, "tables": _tables_plain}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once, each output written once; the multiply-adds of the definition."""
    B = case["B"]
    if case["op"] == "tables":
        held, new = _row_tokens(case)
        pages = sum(-(-(a + b) // case["page"]) - a // case["page"] for a, b in zip(held, new))
        return {"bytes": 4 * (sum(new) + 2 * pages + 4 * B), "flops": 4 * sum(new) + 8 * B}
    N, Hk = case["N"], case["Hk"]
    if case["op"] == "step":
        H = case["H"]
        return {"bytes": 8 * B * H * N * N + 4 * B * (Hk + H) * N + 4 * B * H, "flops": 7 * B * H * N * N}
    if case["op"] == "delta":
        H, n = case["H"], B * case["T"]
        per = 2 * (2 * Hk + 2 * H) * N + 4 * H                   # q, k, v, y, g, beta
        states = 4 * B * H * N * N
        if case["train"]:                                        # and dy, dq, dk, dv, dg, dbeta
            return {"bytes": n * (per + 2 * (2 * Hk + 2 * H) * N + 4 * H) + states * (4 if case["state"] else 1) + (4 * n if case["docs"] else 0), "flops": 21 * n * H * N * N}
        return {"bytes": n * per + states * (2 if case["state"] else 1) + (4 * n if case["docs"] else 0), "flops": 7 * n * H * N * N}
    if case["op"] == "write":
        held, new = _row_tokens(case)
        n, pages = sum(new), sum(-(-(a + b) // case["page"]) - a // case["page"] for a, b in zip(held, new))
        return {"bytes": 2 * n * Hk * N * 3 + 16 * pages * Hk + 4 * n, "flops": 4 * n * Hk * N}
    H, lens = case["H"], _spread(case["longest"], B)
    pages = sum(-(-n // case["page"]) for n in lens)
    return {"bytes": 2 * sum(lens) * Hk * N + 8 * pages * Hk + 4 * pages + 4 * B + 4 * B * H * N, "flops": 4 * sum(lens) * H * N}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"step": _step_exact, "delta": _delta_exact, "write": _write_exact, "paged8": _paged8_exact, "tables": _tables_exact}[case["op"]](state)


def _step_exact(state):
    H, Hk, N = (state["case"][n] for n in ("H", "Hk", "N"))
    head = torch.arange(H, device=DEV) * Hk // H
    q, k, v, g, beta, s = (state[n].double() for n in ("q", "k", "v", "g", "beta", "s0"))
    s = g.exp()[:, :, None, None] * s
    k = k[:, head, :, None]
    s = s + beta[:, :, None, None] * k * (v[:, :, None, :] - (k * s).sum(2, keepdim=True))
    return [(q[:, head, :, None] * s).sum(2) / math.sqrt(N), s]


def _delta_exact(state):
    """Token by token, and back again, the states of 64 tokens at a time made anew on the way back."""
    case = state["case"]
    B, T, H, Hk, N = (case[n] for n in ("B", "T", "H", "Hk", "N"))
    if T > 8192 and case["train"]:
        return None
    head = torch.arange(H, device=DEV) * Hk // H
    token = lambda n, t: state[n][:, t].detach().double()
    root = 1 / math.sqrt(N)
    doc = state["doc"]

    def forward(s, t):
        """The state after token t, what entered its update, and the update."""
        a = token("g", t).exp()
        if doc is not None:
            if t > 0:
                a = torch.where((doc[:, t] != doc[:, t - 1])[:, None], torch.zeros_like(a), a)
            a = torch.where((doc[:, t] < 0)[:, None], torch.ones_like(a), a)
        k = token("k", t)[:, head]
        d = a[:, :, None, None] * s
        u = token("v", t) - torch.matmul(k.unsqueeze(2), d).squeeze(2)
        w = token("beta", t)[:, :, None] * u
        if doc is not None:
            w = w * (doc[:, t] >= 0)[:, None, None]
        return a, d, u, torch.addcmul(d, k.unsqueeze(3), w.unsqueeze(2))

    s = torch.zeros(B, H, N, N, device=DEV, dtype=torch.float64) if state["s0"] is None else state["s0"].detach().double()
    y = torch.empty(B, T, H, N, device=DEV, dtype=torch.float64)
    kept = []
    for t in range(T):
        if t % 64 == 0 and case["train"]:
            kept.append(s)
        s = forward(s, t)[3]
        y[:, t] = torch.matmul(token("q", t)[:, head].unsqueeze(2), s).squeeze(2) * root
    alive = None if doc is None else (doc >= 0).double()[:, :, None, None]
    out = [y if alive is None else y * alive, s]
    if not case["train"]:
        return out
    dq, dk = (torch.zeros(B, T, Hk, N, device=DEV, dtype=torch.float64) for _ in range(2))
    dv = torch.empty_like(y)
    dg, db = (torch.empty(B, T, H, device=DEV, dtype=torch.float64) for _ in range(2))
    ds = torch.zeros_like(s) if state["s0"] is None else state["dsT"].double()
    for lo in range((T - 1) // 64 * 64, -1, -64):
        states = [kept.pop()]
        for t in range(lo, min(T, lo + 64)):
            states.append(forward(states[-1], t)[3])
        for t in range(min(T, lo + 64) - 1, lo - 1, -1):
            live = 1.0 if doc is None else (doc[:, t] >= 0).double()[:, None, None]
            before, after = states[t - lo], states[t - lo + 1]
            a, d, u, _ = forward(before, t)
            q, k, b = token("q", t)[:, head], token("k", t)[:, head], token("beta", t)[:, :, None]
            o = token("dy", t) * root * live
            dq.index_put_((torch.arange(B, device=DEV)[:, None], torch.tensor(t, device=DEV), head[None, :]), torch.matmul(after, o.unsqueeze(3)).squeeze(3), accumulate=True)
            ds = torch.addcmul(ds, q.unsqueeze(3), o.unsqueeze(2))
            dw = torch.matmul(k.unsqueeze(2), ds).squeeze(2) * live
            w = b * u * live
            du = b * dw
            dv[:, t] = du
            db[:, t] = (dw * u).sum(2)
            mine = torch.matmul(ds, w.unsqueeze(3)).squeeze(3) - torch.matmul(d, du.unsqueeze(3)).squeeze(3)
            dk.index_put_((torch.arange(B, device=DEV)[:, None], torch.tensor(t, device=DEV), head[None, :]), mine, accumulate=True)
            ds = torch.addcmul(ds, k.unsqueeze(3), du.unsqueeze(2), value=-1)
            slope = (ds * d).sum((2, 3))
            dg[:, t] = slope if doc is None else slope * live[:, :, 0]
            ds = a[:, :, None, None] * ds
    out += [dq, dk, dv, dg, db]
    return out + [ds] if state["s0"] is not None else out


def _rounded8(x):
    """To the nearest number of four significant bits, ties to even ones; the step stays 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _write_exact(state):
    """Page by page in the order of their numbers: all the new tokens of a page side by side."""
    case = state["case"]
    page = case["page"]
    slots = state["slots"].long()
    touched, which = torch.unique(slots // page, return_inverse=True)
    here = torch.zeros(touched.shape[0], page, dtype=torch.bool, device=DEV)
    here[which, slots % page] = True
    begin = torch.where(here, torch.arange(page, device=DEV), page).amin(1)
    codes, factors = [], []
    for x, pages, scales in ((state["k"], state["k_pages"], state["k_scales"]), (state["v"], state["v_pages"], state["v_scales"])):
        all_pages, all_scales = pages.double(), scales.double()
        new = torch.zeros(touched.shape[0], page, *x.shape[1:], dtype=torch.float64, device=DEV)
        new[which, slots % page] = x.double()
        top = new.abs().amax((1, 3))
        fit = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-100.0))
        scale = torch.where((begin > 0)[:, None], torch.maximum(fit, all_scales[touched]), fit)
        old = (torch.arange(page, device=DEV)[None, :] < begin[:, None])[:, :, None, None]
        was = all_pages[touched]
        now = torch.where(old, _rounded8(was * (all_scales[touched] / scale)[:, None, :, None]), was)
        now = torch.where(here[:, :, None, None], _rounded8(new / scale[:, None, :, None]), now)
        all_pages[touched], all_scales[touched] = now, scale
        codes.append(all_pages)
        factors.append(all_scales)
    return codes + factors


def _paged8_exact(state):
    case = state["case"]
    H, Hk, N, page = case["H"], case["Hk"], case["N"], case["page"]
    y = torch.empty(case["B"], H, N, device=DEV, dtype=torch.float64)
    kp, vp = (state[n].view(torch.uint8) for n in ("k_pages", "v_pages"))
    for b, n in enumerate(state["lens"].tolist()):
        at = torch.arange(n, device=DEV)
        spots = state["table"][b].long()[at // page]
        for h in range(Hk):
            k = kp[spots, at % page, h].view(FP8).double() * state["k_scales"][spots, h].double()[:, None]
            v = vp[spots, at % page, h].view(FP8).double() * state["v_scales"][spots, h].double()[:, None]
            mine = slice(h * (H // Hk), (h + 1) * (H // Hk))
            s = (state["q"][b, mine].double() @ k.transpose(0, 1)) / math.sqrt(N)
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if state["slopes"] is not None:
                s = s - state["slopes"][mine].double()[:, None] * (n - 1 - at)[None, :].double()
            y[b, mine] = torch.softmax(s, 1) @ v
    return [y]


def _tables_exact(state):
    return None
