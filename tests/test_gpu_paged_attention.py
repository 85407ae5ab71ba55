"""GPU: attention of one new token over a paged cache against its 64-bit definition, with bounds element by element."""
import pytest
import torch

from oracle import mixers as O
from rwkv_cuda_amd import attention, paged_attention as PA
from _gpu_util import DEV
from _mixers_util import DT, graph_of, randn, within

pytestmark = pytest.mark.gpu


def cache(lens, H, Hk, N, page, dt, seed=0, spare=3):
    """q, pages in a shuffled order with some unused ones full of NaN, and NaN behind each sequence's last token."""
    B, need = len(lens), [max(0, -(-n // page)) for n in lens]
    P = sum(need) + spare
    M = max(max(need), 1) + 1
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(P, generator=g)
    kp, vp = (randn(P, page, Hk, N, seed=seed + i).to(dt) for i in (1, 2))
    table = torch.full((B, M), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
        if lens[b] > 0 and lens[b] % page:
            for z in (kp, vp):
                z[table[b, n - 1], lens[b] % page:] = float("nan")
    for z in (kp, vp):
        z[order[at:]] = float("nan")
    return [z.to(DEV) for z in (randn(B, H, N, seed=seed + 3).to(dt), kp, vp, table, torch.tensor(lens, dtype=torch.int32))]


def check(q, kp, vp, table, lens, **how):
    y = PA.RUN_CUDA(q, kp, vp, table, lens, **how)
    torch.cuda.synchronize()
    within("y", y, O.paged_attention(q, kp, vp, table, lens, **how)["y"])
    return y


LENS = [[1], [0, 3, 64], [1, 2, 15, 16, 17, 31, 33], [63, 64, 65, 127, 128, 129], [1000, 5, -4, 257], [4097, 1, 2048]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("H,Hk,N,dtype", [(4, 4, 64, "bf16"), (8, 2, 128, "fp16"), (16, 1, 128, "bf16"), (6, 2, 80, "bf16"), (40, 1, 64, "fp16"), (3, 3, 8, "bf16")])
@pytest.mark.parametrize("page", [1, 16, 256])
def test_against_the_definition(lib, lens, H, Hk, N, dtype, page):
    print(f"\n{lens} {H} {Hk} {N} {dtype} {page}", flush=True)
    check(*cache(lens, H, Hk, N, page, DT[dtype]))


@pytest.mark.parametrize("H,Hk,N,B", [(32, 32, 64, 17), (40, 8, 40, 64), (136, 8, 64, 35)])
def test_many_heads(lib, H, Hk, N, B):
    """Workgroups enough to be dealt out by eights of neighbouring heads, their number no multiple of the XCDs'; also with heads in chunks."""
    lens = torch.randint(0, 300, (B,), generator=torch.Generator().manual_seed(H)).tolist()
    check(*cache(lens, H, Hk, N, 16, torch.bfloat16, seed=61))


@pytest.mark.parametrize("how", ["cap", "bias", "both", "scale"])
def test_caps_and_biases(lib, how):
    H = 8
    o = dict(cap=3.0) if how in ("cap", "both") else {}
    if how in ("bias", "both"):
        o["slopes"] = torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)
    if how == "scale":
        o["scale"] = 2.0
    for dt in (torch.bfloat16, torch.float16):
        check(*cache([5, 700, 77, 2000], H, 2, 64, 32, dt, seed=5), **o)


def test_it_is_the_last_row_of_attention(lib):
    """One sequence through both operators, the cache as pages in order."""
    T, H, Hk, N = 333, 8, 2, 64
    q, k, v = (randn(1, T, h, N, seed=i).to(torch.bfloat16).to(DEV) for i, h in enumerate((H, Hk, Hk)))
    slopes = torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)
    want = attention.RUN_CUDA(q, k, v, slopes=slopes, cap=10.0)[:, -1]
    pad = torch.zeros(1, 352 - T, Hk, N, device=DEV, dtype=torch.bfloat16)
    kp, vp = (torch.cat([z, pad], 1).view(-1, 32, Hk, N) for z in (k, v))
    table = torch.arange(11, dtype=torch.int32, device=DEV).view(1, 11)
    got = PA.RUN_CUDA(q[:, -1], kp, vp, table, torch.tensor([T], dtype=torch.int32, device=DEV), slopes=slopes, cap=10.0)
    value, bound = O.attention(q[:, -1:], k, v, slopes=slopes, cap=10.0)["y"]
    within("paged", got, (value[:, 0], bound[:, 0]))
    within("attention", want, (value[:, 0], bound[:, 0]))


@pytest.mark.parametrize("H,Hk,N", [(8, 2, 128), (2, 2, 64), (24, 1, 40)])
def test_the_new_token_is_written_and_seen(lib, H, Hk, N):
    """Token by token from an empty cache of NaN, several sequences of different lengths; nothing else of the cache changes."""
    B, page, M = 3, 16, 6
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(B * M, generator=g).view(B, M).to(torch.int32).to(DEV)
    kp, vp = (torch.full((B * M, page, Hk, N), float("nan"), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    kw, vw = kp.clone(), vp.clone()
    start = [0, 13, 40]
    for b, n in enumerate(start):
        for t in range(n):
            for z, w in ((kp, kw), (vp, vw)):
                z[table[b, t // page], t % page] = w[table[b, t // page], t % page] = randn(Hk, N, seed=1000 * b + t).to(torch.bfloat16).to(DEV)
    for step in range(20):
        lens = torch.tensor([n + step + 1 for n in start], dtype=torch.int32, device=DEV)
        q, k, v = (randn(B, h, N, seed=5000 + 3 * step + i).to(torch.bfloat16).to(DEV) for i, h in enumerate((H, Hk, Hk)))
        y = PA.RUN_CUDA(q, kp, vp, table, lens, k=k, v=v)
        for b in range(B):
            t = int(lens[b]) - 1
            kw[table[b, t // page], t % page], vw[table[b, t // page], t % page] = k[b], v[b]
        torch.cuda.synchronize()
        assert torch.equal(kp.view(torch.int16), kw.view(torch.int16)) and torch.equal(vp.view(torch.int16), vw.view(torch.int16))
        within("y", y, O.paged_attention(q, kw, vw, table, lens)["y"])
        assert torch.equal(y, PA.RUN_CUDA(q, kp, vp, table, lens))


def test_pages_that_are_not_there_are_left_out(lib):
    """Numbers below 0 and from P on, in the middle and at the end, and more tokens than the table has pages for: nothing is read or
    written there.  A sequence none of whose pages is there has y = 0."""
    q, kp, vp, table, lens = cache([300, 100, 60, 40], 4, 2, 64, 16, torch.bfloat16, seed=9)
    kp, vp = (torch.nan_to_num(z) for z in (kp, vp))                 # the last sequence sees the first one's pages to their ends
    P = kp.shape[0]
    table[0, 3], table[0, 7], table[1, -1] = -1, P, 2 ** 31 - 1
    table[2, :] = -2 ** 31
    lens[3] = 16 * table.shape[1] + 50
    table[3] = table[0]
    kept = kp.clone()
    k, v = (randn(4, 2, 64, seed=i).to(torch.bfloat16).to(DEV) for i in (1, 2))
    y = check(q, kp, vp, table, lens)
    assert not y[2].any()
    table[0, 18] = P + 5                                             # the page of the new token
    lens[1] = 0
    y = PA.RUN_CUDA(q, kp, vp, table, lens, k=k, v=v)
    torch.cuda.synchronize()
    assert torch.equal(kp.view(torch.int16), kept.view(torch.int16)) and not y[1:3].any()
    within("y", y, O.paged_attention(q, kp, vp, table, lens)["y"])


def test_views_of_one_cache_and_shared_pages(lib):
    """Keys and values in one tensor, heads first in a page; sequences that share their first pages."""
    lens, H, Hk, N, page = [200, 190, 64], 8, 2, 64, 16
    q, kp, vp, table, lens = cache(lens, H, Hk, N, page, torch.bfloat16, seed=11)
    table[1, :8] = table[0, :8]
    table[2, :4] = table[0, :4]
    both = torch.stack([kp, vp], 1)
    y = check(q, kp, vp, table, lens)
    assert torch.equal(y, PA.RUN_CUDA(q, both[:, 0], both[:, 1], table, lens))
    first = [z.transpose(1, 2).contiguous().transpose(1, 2) for z in (kp, vp)]
    assert torch.equal(y, PA.RUN_CUDA(q, *first, table, lens))


def test_a_cache_beyond_2_31_elements(lib):
    page, Hk, N = 256, 8, 128
    P = (1 << 31) // (page * Hk * N) + 20
    kp = torch.empty(P, page, Hk, N, device=DEV, dtype=torch.bfloat16)
    vp = torch.empty_like(kp)
    table = torch.tensor([[P - 1, 3, P - 9]], dtype=torch.int32, device=DEV)
    for z, s in ((kp, 1), (vp, 2)):
        z[table[0].long()] = randn(3, page, Hk, N, seed=s).to(torch.bfloat16).to(DEV)
    q = randn(1, 16, N, seed=3).to(torch.bfloat16).to(DEV)
    lens = torch.tensor([700], dtype=torch.int32, device=DEV)
    small = [z[table[0].long()].contiguous() for z in (kp, vp)]
    got = PA.RUN_CUDA(q, kp, vp, table, lens)
    assert torch.equal(got, check(q, *small, torch.arange(3, dtype=torch.int32, device=DEV).view(1, 3), lens))


def test_captured_and_replayed(lib):
    """A graph that decodes: lengths, table and inputs change between the replays."""
    q, kp, vp, table, lens = cache([900, 30, 511], 8, 2, 128, 16, torch.bfloat16, seed=13)
    kp, vp = (torch.nan_to_num(z) for z in (kp, vp))
    k, v = (randn(3, 2, 128, seed=i).to(torch.bfloat16).to(DEV) for i in (1, 2))
    run = lambda: PA.RUN_CUDA(q, kp, vp, table, lens, k=k, v=v)
    (g1, o1), (g2, o2) = graph_of(run), graph_of(run)
    for i in range(4):
        lens.copy_(torch.tensor([900 - 17 * i, 20 + i, 500 + i], dtype=torch.int32))
        q.copy_(randn(*q.shape, seed=40 + i).to(q.dtype))
        want = run().clone()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, o1) and torch.equal(want, o2)


def test_a_row_is_what_it_is_alone_and_the_same_every_time(lib):
    q, kp, vp, table, lens = cache([3000, 20, 1500], 8, 2, 64, 64, torch.float16, seed=15)
    y = PA.RUN_CUDA(q, kp, vp, table, lens)
    for _ in range(3):
        assert torch.equal(y, PA.RUN_CUDA(q, kp, vp, table, lens))
