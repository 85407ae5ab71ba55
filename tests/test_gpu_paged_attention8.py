"""GPU: the paged cache in 8 bits, bit by bit against its definition, and the attention over it, element by element."""
import pytest
import torch

from oracle import mixers as O
from rwkv_cuda_amd import paged_attention as PA, paged_attention8 as P8
from _cache8_util import F8, rounded, values, write
from _gpu_util import DEV
from _mixers_util import DT, graph_of, randn, within

pytestmark = pytest.mark.gpu
NAN = 0x7f


def pool(P, page, Hk, N, seed=0, fill=None):
    """Codes and scales of keys and values: drawn, or `fill` everywhere."""
    out = []
    for i in (1, 2):
        z = randn(P, page, Hk, N, seed=seed + i, scale=90.0).clamp(-448, 448).to(F8) if fill is None else torch.full((P, page, Hk, N), fill, dtype=torch.uint8).view(F8)
        out.append(z.to(DEV))
    g = torch.Generator().manual_seed(seed)
    return out + [torch.exp2(torch.randint(-9, -4, (P, Hk), generator=g).float()).to(DEV) for _ in range(2)]


def same(cache, want):
    torch.cuda.synchronize()
    for pages, scales, (codes, factors) in ((cache[0], cache[2], want[0]), (cache[1], cache[3], want[1])):
        assert torch.equal(scales.double().cpu(), factors)
        got = pages.float().double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(codes)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes))


def put(k, v, cache, slots):
    """WRITE, held to the definition."""
    want = [write(x, cache[i], cache[i + 2], slots) for i, x in ((0, k), (1, v))]
    P8.WRITE(k, v, *cache, slots)
    same(cache, want)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_every_code_and_every_rounding(lib):
    """All finite bf16 numbers of 16 binades, and all codes rounded again by every step."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits[torch.isfinite(bits.float()) & (bits.float().abs() <= 448) & ((bits.float().abs() >= 2.0 ** -14) | (bits.float() == 0))]
    n = x.numel() // 16 * 16
    x = x[:n].view(-1, 1, 16)
    x = torch.cat([x, torch.full((x.shape[0], 1, 16), 448.0, dtype=torch.bfloat16)], 2).to(DEV)        # a scale of 1
    cache = pool(x.shape[0], 1, 1, 32, fill=0)
    P8.WRITE(x, x, *cache, torch.arange(x.shape[0], dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert bool((cache[2] == 1).all()) and torch.equal(cache[0].float().double()[:, 0], rounded(x.double()))
    codes = torch.arange(256, dtype=torch.uint8).view(1, 16, 16)
    codes[codes.view(F8).float().isnan()] = 0
    for by in range(0, 20):
        cache = [torch.zeros(1, 32, 1, 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
        for z in cache:
            z[0, :16, 0] = codes.to(DEV)
        cache = [z.view(F8) for z in cache] + [torch.ones(1, 1, device=DEV) for _ in range(2)]
        new = torch.full((1, 1, 16), 448.0 * 2.0 ** by, device=DEV).to(torch.bfloat16)
        put(new, new, cache, i32([16]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hk,N,page", [(1, 16, 1), (2, 64, 16), (3, 80, 4), (8, 128, 64), (1, 112, 256), (33, 32, 2)])
def test_writing(lib, dtype, Hk, N, page):
    """Runs of all lengths, from empty pages and behind tokens; pages in no order; slots outside the cache."""
    P = 12
    g = torch.Generator().manual_seed(N)
    for case in range(3):
        cache = pool(P, page, Hk, N, seed=N + case)
        slots = []
        for p in torch.randperm(P, generator=g).tolist()[:8]:
            lo = int(torch.randint(0, page, (1,), generator=g)) if case else 0
            hi = int(torch.randint(lo, page, (1,), generator=g)) + 1
            slots += list(range(p * page + lo, p * page + hi))
            if case == 2:
                slots += [-1, P * page, 2 ** 31 - 1, -2 ** 31][:int(torch.randint(0, 5, (1,), generator=g))]
        n = len(slots)
        k, v = (randn(n, Hk, N, seed=7 * case + i, scale=(0.1, 3.0, 1000.0)[case]).to(DT[dtype]).to(DEV) for i in (3, 4))
        put(k, v, cache, i32(slots))


def test_many_tokens_at_once(lib):
    """Enough for a wave to look through several tokens; pages that end inside of what it looks through, and runs beyond it."""
    page, Hk, N, B = 32, 4, 64, 9
    lens = [900, 1, 33, 31, 64, 700, 500, 65, 1200]
    need = [-(-n // page) for n in lens]
    P = sum(need)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(1)).tolist()
    slots, at = [], 0
    for n, m in zip(lens, need):
        skip = 5 if n > 40 else 0                                # the first page holds five tokens
        slots += [order[at + t // page] * page + t % page for t in range(skip, n)]
        at += m
    k, v = (randn(len(slots), Hk, N, seed=i).to(torch.bfloat16).to(DEV) for i in (1, 2))
    cache = pool(P, page, Hk, N, seed=3)
    put(k, v, cache, i32(slots))
    again = [z.clone() for z in cache]                           # the same tokens once more: nothing changes
    P8.WRITE(k, v, *cache, i32(slots))
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, again))


def test_values_at_their_ends(lib):
    """Zeros, the least and the largest numbers, infinities and NaN: the scale goes by what is finite."""
    top = torch.finfo(torch.bfloat16).max
    rows = [[0.0] * 16, [top] + [1.0] * 15, [float("inf"), -2.0] + [0.5] * 14, [float("nan")] * 16, [1e-38] * 16, [-top] * 16, [2.0 ** -100, -448 * 2.0 ** -100] + [0.0] * 14, [448.0, 449.0] * 8, [-0.0] * 16]
    k = torch.tensor(rows, dtype=torch.float32).to(torch.bfloat16).view(-1, 1, 16).to(DEV)
    cache = pool(len(rows), 4, 1, 16, seed=5)
    put(k, k.flip(0), cache, i32([4 * i for i in range(len(rows))]))
    cache = pool(len(rows), 4, 1, 16, seed=5)
    put(k, k.flip(0), cache, i32([4 * i + 2 for i in range(len(rows))]))


def test_written_views_and_nothing_else(lib):
    """Keys and values in one tensor, heads first in a page, tokens as views of a projection; bytes between them stay."""
    P, page, Hk, N, n = 6, 16, 2, 32, 40
    qkv = randn(n, 3 * Hk * N + 8, seed=1).to(torch.bfloat16).to(DEV)[:, 8:]
    k, v = (z.unflatten(1, (Hk, N)) for z in (qkv[:, Hk * N:2 * Hk * N], qkv[:, 2 * Hk * N:]))
    slots = i32(list(range(3, 43)))
    plain = pool(P, page, Hk, N, seed=2)
    both = torch.full((P, Hk, 2, page, N + 16), 0x55, dtype=torch.uint8, device=DEV)
    views = [both[:, :, i, :, :N].transpose(1, 2) for i in (0, 1)]
    for z, w in zip(views, plain):
        z.copy_(w.view(torch.uint8))
    cache = [z.view(F8) for z in views] + [z.clone() for z in plain[2:]]
    put(k, v, plain, slots)
    P8.WRITE(k, v, *cache, slots)
    torch.cuda.synchronize()
    assert all(torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, plain)) and bool((both[..., N:] == 0x55).all())
    q = randn(1, 4, N, seed=5).to(torch.bfloat16).to(DEV)
    table, lens = torch.arange(P, dtype=torch.int32, device=DEV).view(1, P), i32([43])
    assert torch.equal(P8.RUN_CUDA(q, *cache, table, lens), P8.RUN_CUDA(q, *plain, table, lens))


def test_no_tokens(lib):
    cache = pool(3, 4, 1, 16, seed=1)
    kept = [z.clone() for z in cache]
    none = torch.empty(0, 1, 16, dtype=torch.bfloat16, device=DEV)
    P8.WRITE(none, none, *cache, i32([]))
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, kept))


# ------------------------------------------------------------------------------------------------ attention
def cache(lens, H, Hk, N, page, dt, seed=0, spare=3):
    """q, a cache whose pages are in a shuffled order, some unused and full of NaN with a scale of NaN, and NaN behind each sequence's last token."""
    B, need = len(lens), [max(0, -(-n // page)) for n in lens]
    P, M = sum(need) + spare, max(max(need), 1) + 1
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed))
    kp, vp, ks, vs = pool(P, page, Hk, N, seed)
    table = torch.full((B, M), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
        if lens[b] > 0 and lens[b] % page:
            for z in (kp, vp):
                z.view(torch.uint8)[table[b, n - 1], lens[b] % page:] = NAN
    for z in (kp, vp):
        z.view(torch.uint8)[order[at:].to(DEV)] = NAN
    for z in (ks, vs):
        z[order[at:].to(DEV)] = float("nan")
    return randn(B, H, N, seed=seed + 3).to(dt).to(DEV), [kp, vp, ks, vs], table.to(DEV), i32(lens)


def check(q, kv, table, lens, **how):
    y = P8.RUN_CUDA(q, *kv, table, lens, **how)
    torch.cuda.synchronize()
    within("y", y, O.paged_attention(q, values(kv[0], kv[2]), values(kv[1], kv[3]), table, lens, **how)["y"])
    return y


LENS = [[1], [0, 3, 64], [1, 2, 15, 16, 17, 31, 33], [63, 64, 65, 127, 128, 129], [1000, 5, -4, 257], [4097, 1, 2048]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("H,Hk,N,dtype", [(4, 4, 64, "bf16"), (8, 2, 128, "fp16"), (16, 1, 128, "bf16"), (6, 2, 80, "bf16"), (40, 1, 64, "fp16"), (3, 3, 16, "bf16")])
@pytest.mark.parametrize("page", [1, 16, 256])
def test_against_the_definition(lib, lens, H, Hk, N, dtype, page):
    print(f"\n{lens} {H} {Hk} {N} {dtype} {page}", flush=True)
    check(*cache(lens, H, Hk, N, page, DT[dtype]))


@pytest.mark.parametrize("H,Hk,N,B", [(32, 32, 64, 17), (40, 8, 48, 64), (136, 8, 64, 35), (16, 16, 128, 40)])
def test_many_heads(lib, H, Hk, N, B):
    lens = torch.randint(0, 300, (B,), generator=torch.Generator().manual_seed(H)).tolist()
    check(*cache(lens, H, Hk, N, 16, torch.bfloat16, seed=61))


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("N,page,dtype", [(64, 16, "bf16"), (128, 8, "fp16"), (48, 2, "fp16"), (112, 128, "bf16")])
def test_query_heads_of_a_key_head(lib, G, N, page, dtype):
    """Each way to lay heads and tokens over the lanes, with caps and biases, over several rounds of the waves; pages missing in the middle of a tile."""
    q, kv, table, lens = cache([1500, 3, 260, 0, 63], 3 * G, 3, N, page, DT[dtype], seed=G)
    for i in range(3, 1500 // page, 5):
        table[0, i] = -1
    check(q, kv, table, lens, cap=20.0, slopes=torch.exp2(-torch.arange(1.0, 3 * G + 1) / G).to(DEV))
    check(q, kv, table, lens)


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


def test_scales_far_apart(lib):
    """Values a million times larger in some pages than in others, and pages of zeros at the least scale: weights keep to their 16 bits."""
    for dt in (torch.bfloat16, torch.float16):
        q, kv, table, lens = cache([700, 90, 2000], 8, 2, 64, 16, dt, seed=6)
        kv[3] *= torch.exp2(torch.randint(-10, 11, kv[3].shape, generator=torch.Generator().manual_seed(1)).float()).to(DEV)
        kv[1].view(torch.uint8)[table[0, 3]] = 0
        kv[3][table[0, 3].long()] = 2.0 ** -100
        check(q, kv, table, lens)


def test_as_paged_attention_where_16_bits_hold_the_values(lib):
    q, kv, table, lens = cache([300, 20, 1500], 8, 2, 64, 16, torch.bfloat16, seed=8)
    kp, vp = (values(kv[i], kv[i + 2]).to(torch.bfloat16) for i in (0, 1))
    want = O.paged_attention(q, values(kv[0], kv[2]), values(kv[1], kv[3]), table, lens)["y"]
    within("16 bits", PA.RUN_CUDA(q, kp, vp, table, lens), want)
    within("8 bits", P8.RUN_CUDA(q, *kv, table, lens), want)


def test_pages_that_are_not_there_are_left_out(lib):
    q, kv, table, lens = cache([300, 100, 60, 40], 4, 2, 64, 16, torch.bfloat16, seed=9)
    for z in kv[:2]:
        z.view(torch.uint8)[z.float().isnan()] = 0
    P = kv[0].shape[0]
    table[0, 3], table[0, 7], table[1, -1] = -1, P, 2 ** 31 - 1
    table[2, :] = -2 ** 31
    lens[3] = 16 * table.shape[1] + 50
    table[3] = table[0]
    y = check(q, kv, table, lens)
    assert not y[2].any()


def test_a_cache_beyond_2_31_bytes(lib):
    page, Hk, N = 256, 8, 128
    P = (1 << 32) // (page * Hk * N) + 20
    kp = torch.empty(P, page, Hk, N, device=DEV, dtype=torch.uint8).view(F8)
    vp = torch.empty_like(kp)
    ks, vs = (torch.full((P, Hk), 2.0 ** -7, device=DEV) for _ in range(2))
    table = i32([[P - 1, 3, P - 9]])
    rows = table[0].long()
    k, v = (randn(600, Hk, N, seed=s).to(torch.bfloat16).to(DEV) for s in (1, 2))
    slots = torch.cat([table[0, i] * page + torch.arange(n, dtype=torch.int32, device=DEV) for i, n in enumerate((256, 256, 88))])
    assert int(slots.max()) * Hk * N > 1 << 31
    P8.WRITE(k, v, kp, vp, ks, vs, slots)
    small = [torch.zeros(3, page, Hk, N, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2)] + [torch.full((3, Hk), 2.0 ** -7, device=DEV) for _ in range(2)]
    put(k, v, small, torch.arange(600, dtype=torch.int32, device=DEV))
    q, lens = randn(1, 16, N, seed=3).to(torch.bfloat16).to(DEV), i32([600])
    got = P8.RUN_CUDA(q, kp, vp, ks, vs, table, lens)
    assert torch.equal(got, check(q, small, i32([[0, 1, 2]]), lens)) and torch.equal(ks[rows], small[2])


def test_captured_and_replayed(lib):
    """A graph that writes a token and decodes: tokens, slots, lengths and table change between the replays; each replay is the eager call."""
    q, kv, table, lens = cache([900, 30, 511], 8, 2, 128, 16, torch.bfloat16, seed=13)
    for z in kv[:2]:
        z.view(torch.uint8)[z.float().isnan()] = 0
    k, v = (randn(3, 2, 128, seed=i).to(torch.bfloat16).to(DEV) for i in (1, 2))
    slots = (table[torch.arange(3), (lens.long() - 1) // 16] * 16 + (lens - 1) % 16).to(torch.int32)

    def step():
        P8.WRITE(k, v, *kv, slots)
        return P8.RUN_CUDA(q, *kv, table, lens)
    (g1, o1), (g2, o2) = graph_of(step), graph_of(step)
    start = [z.clone() for z in kv]
    for i in range(4):
        lens.copy_(torch.tensor([900 - 17 * i, 20 + i, 500 + i], dtype=torch.int32))
        slots.copy_(table[torch.arange(3), (lens.long() - 1) // 16] * 16 + (lens - 1) % 16)
        k.copy_(randn(*k.shape, seed=40 + i, scale=1 + i).to(k.dtype))
        results = []
        for call in (step, g1.replay, g2.replay):
            for z, s in zip(kv, start):
                z.copy_(s)
            y = call()
            torch.cuda.synchronize()
            results.append([(y if call is step else o1 if call == g1.replay else o2).clone()] + [z.clone().view(torch.uint8) for z in kv])
        for r in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(results[0], r)), i


def test_versions_and_streams(lib):
    """What is written finds out; two streams at once write and read caches of their own."""
    caches = [pool(20, 16, 2, 64, seed=s) for s in (1, 2)]
    k, v = (randn(300, 2, 64, seed=s).to(torch.bfloat16).to(DEV) for s in (3, 4))
    slots = torch.arange(300, dtype=torch.int32, device=DEV)
    q, table, lens = randn(1, 4, 64, seed=5).to(torch.bfloat16).to(DEV), torch.arange(20, dtype=torch.int32, device=DEV).view(1, 20), i32([300])
    before = [z._version for z in caches[0]]
    want = []
    for c in caches:
        d = [z.clone() for z in c]
        P8.WRITE(k, v, *d, slots)
        want.append(P8.RUN_CUDA(q, *d, table, lens))
    torch.cuda.synchronize()
    got = []
    for c, s in zip(caches, [torch.cuda.Stream() for _ in caches]):
        with torch.cuda.stream(s):
            P8.WRITE(k, v, *c, slots)
            got.append(P8.RUN_CUDA(q, *c, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(z._version > b for z, b in zip(caches[0], before))


@pytest.mark.parametrize("H,Hk,N,lens", [(4, 4, 64, [3000, 0, 70]), (8, 2, 128, [2500, 1]), (16, 2, 64, [4000]), (32, 2, 128, [1300, 77])])
def test_what_memory_held_before_counts_nowhere(lib, H, Hk, N, lens):
    """The same bits whatever the output's and the workspace's memory held, and again."""
    q, kv, table, lens = cache(lens, H, Hk, N, 16, torch.bfloat16, seed=21)
    want = check(q, kv, table, lens)
    for value in [0.0, float("nan"), 1e4] + 10 * [None]:
        if value is not None:
            held = [torch.full((n,), value, device=DEV) for n in (1 << 8, 1 << 12, 1 << 16, 1 << 18, 1 << 20) for _ in range(12)]
            torch.cuda.synchronize()
            del held
        assert torch.equal(P8.RUN_CUDA(q, *kv, table, lens), want), value


@pytest.mark.parametrize("H,Hk,N", [(8, 2, 64), (4, 4, 128), (32, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("M", [8, 70, 500])
def test_scales_as_far_apart_as_there_are(lib, H, Hk, N, M):
    """Pages of zeros at the least scale beside pages at scales up to 2^110, in one wave and in several, one after the other either way round: every token keeps its share of the softmax's sum."""
    page, n = 16, 16 * M - 3
    for small_first in (True, False):
        for big in (27.0, 60.0, 110.0):
            q, kv, table, lens = cache([n, n // 2], H, Hk, N, page, torch.bfloat16, seed=M)
            for b in range(2):
                pages = table[b, :-(-int(lens[b]) // page)].long()
                kv[3][pages] = 2.0 ** big
                zeros = pages[:len(pages) // 2] if small_first else pages[len(pages) // 2:]
                kv[1].view(torch.uint8)[zeros] = 0
                kv[3][zeros] = 2.0 ** -100
            print(f"\nscales 2^-100 and 2^{big}, {'small' if small_first else 'large'} ones first", flush=True)
            check(q, kv, table, lens)
            check(q, kv, table, lens, cap=20.0, slopes=torch.exp2(-torch.arange(1.0, H + 1)).to(DEV))
