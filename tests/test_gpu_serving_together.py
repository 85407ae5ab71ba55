"""GPU: the gated delta rule, the page tables and the cache in 8 bits as a hybrid model uses them: a layer of the delta rule, then one of attention, on packed
documents in training, and in serving prompts of several lengths and then token by token, captured."""
import pytest
import torch

from oracle import delta as OD, mixers as OM
from rwkv_cuda_amd import attention as A, gated_delta as G, page_tables as PT, paged_attention8 as P8
from _cache8_util import F8, values, write
from _delta_util import inputs, near
from _gpu_util import DEV
from _mixers_util import DT, doc_ids, graph_of, randn, within

pytestmark = pytest.mark.gpu
H, HK, N = 8, 2, 64


def heads(z):
    """The delta layer's output as queries, and its first heads as keys and values."""
    return z, z[..., :HK, :], z[..., HK:2 * HK, :]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,T,kind", [(2, 200, "two"), (3, 90, "padded"), (1, 1, "two")])
def test_training_on_packed_documents(lib, dtype, B, T, kind):
    t, _, dy, _ = inputs(B, T, H, HK, N, DT[dtype], seed=1)
    doc = doc_ids(B, T, kind, seed=2).to(DEV)
    leaves = [z.requires_grad_(True) for z in t]
    z, _ = G.RUN_CUDA(*leaves, doc=doc)
    z.retain_grad()
    y = A.RUN_CUDA(*heads(z), doc=doc)
    grads = torch.autograd.grad(y, [z, *leaves], dy)
    want = OM.attention(*heads(z.detach()), doc=doc, dy=dy)
    within("y", y, want["y"])
    want = OD.gated_delta(*t, doc=doc, dy=grads[0])
    near("z", z, want["y"])
    for n, g in zip(("dq", "dk", "dv", "dg", "dbeta"), grads[1:]):
        near(n, g, want[n])


def test_prompts_and_then_token_by_token(lib):
    B, page, M, new, dt = 5, 16, 6, 20, torch.bfloat16
    prompt = [40, 0, 17, 16, 33]
    T = max(prompt)
    t, _, _, _ = inputs(B, T, H, HK, N, dt, seed=5)
    tn, _, _, _ = inputs(B, new, H, HK, N, dt, seed=6)
    doc = torch.where(torch.arange(T) < torch.tensor(prompt)[:, None], 0, -1).to(torch.int32).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    pool, taken, lens = torch.randperm(B * M, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV), i32([0]), i32([0] * B)
    table = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
    cache = [torch.full((B * M, page, HK, N), 0x7f, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2)] + [torch.full((B * M, HK), 1.0, device=DEV) for _ in range(2)]
    with torch.no_grad():
        z, s = G.RUN_CUDA(*t, doc=doc)
        _, k, v = heads(z)
        slots, starts, lens2, taken2 = PT.EXTEND(lens, i32(prompt), table, pool, taken, page, sum(prompt))
        lens.copy_(lens2), taken.copy_(taken2)
        packed = doc.flatten() >= 0
        want = [write(x.flatten(0, 1)[packed], cache[i], cache[i + 2], slots) for i, x in ((0, k), (1, v))]
        P8.WRITE(k.flatten(0, 1)[packed], v.flatten(0, 1)[packed], *cache, slots)
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(torch.nan_to_num(cache[i].float().double().cpu(), nan=999.0), torch.nan_to_num(want[i][0], nan=999.0)) and torch.equal(cache[i + 2].double().cpu(), want[i][1])
        now, one = [x[:, 0].clone() for x in tn], i32([1] * B)

        def step():
            z = G.STEP(*now, s)
            q, k, v = heads(z)
            slots, _, held, out = PT.EXTEND(lens, one, table, pool, taken, page, B)
            lens.copy_(held), taken.copy_(out)
            P8.WRITE(k, v, *cache, slots)
            return z, P8.RUN_CUDA(q, *cache, table, lens)
        kept = [x.clone() for x in (s, lens, taken, table, *cache)]
        graph, (zg, yg) = graph_of(step)
        torch.cuda.synchronize()
        for x, y in zip((s, lens, taken, table, *cache), kept):
            x.copy_(y)
        zs, ys = [], []
        for i in range(new):
            for x, y in zip(now, tn):
                x.copy_(y[:, i])
            graph.replay()
            torch.cuda.synchronize()
            assert lens.tolist() == [n + i + 1 for n in prompt] and int(taken) == sum(-(-int(n) // page) for n in lens)
            zs.append(zg.clone()), ys.append(yg.clone())
            within("y", yg, OM.paged_attention(zg, values(cache[0], cache[2]), values(cache[1], cache[3]), table, lens)["y"])
    for b, n in enumerate(prompt):                               # the delta layer's rows are those of the whole sequences
        whole = [torch.cat([x[b:b + 1, :n], y[b:b + 1]], 1) for x, y in zip(t, tn)]
        want = OD.gated_delta(*whole)
        near("z", torch.stack([x[b] for x in zs]), want["y"][0, n:])
        near("s", s[b], want["sT"][0])
    # ... and what the cache stands for are its keys, to half a step of their code (and of another one where their page's scale grew)
    b = 0
    rows = torch.cat([z[b, :prompt[b]], torch.stack([x[b] for x in zs])])[:, :HK].double()
    at = torch.arange(len(rows), device=DEV)
    got = values(cache[0], cache[2])[table[b].long()[at // page], at % page]
    least = cache[2].double()[table[b].long()[at // page]][..., None] * 2.0 ** -10
    assert bool(((got - rows).abs() <= 2 * (2.0 ** -4 * rows.abs() + least)).all())
