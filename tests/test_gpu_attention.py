"""GPU: attention against its 64-bit definition, with bounds element by element."""
import pytest
import torch

from oracle import mixers as O
from rwkv_cuda_amd import attention as A
from _gpu_util import DEV
from _mixers_util import DT, doc_ids, graph_of, randn, within

pytestmark = pytest.mark.gpu


def inputs(B, Tq, Tk, H, Hk, N, dt, seed=0, scale=1.0):
    return [randn(*s, seed=seed + i, scale=scale).to(dt).to(DEV) for i, s in enumerate([(B, Tq, H, N), (B, Tk, Hk, N), (B, Tk, Hk, N), (B, Tq, H, N)])]


def check(q, k, v, dy, seen=None, **how):
    """`seen`: the tensors that the oracle gets instead of q, k, v."""
    t = [z.detach().requires_grad_(True) for z in (q, k, v)]
    y = A.RUN_CUDA(*t, **how)
    assert y.is_contiguous() and y.dtype == q.dtype
    grads = torch.autograd.grad([y], t, [dy])
    with torch.no_grad():
        assert torch.equal(y, A.RUN_CUDA(q, k, v, **how))
    torch.cuda.synchronize()
    want = O.attention(*(seen or (q, k, v)), dy=dy, **how)
    for n, got in zip(["y", "dq", "dk", "dv"], [y] + list(grads)):
        within(n, got, want[n])


SHAPES = [(1, 1, 1, 1, 1, 64), (2, 1, 70, 2, 1, 64), (1, 2, 2, 2, 2, 128), (2, 31, 31, 2, 1, 64), (1, 32, 33, 4, 1, 128), (2, 64, 64, 1, 1, 64), (1, 65, 65, 3, 3, 64),
          (1, 100, 227, 4, 2, 128), (2, 127, 127, 2, 2, 128), (1, 129, 129, 8, 1, 64), (1, 255, 300, 2, 1, 96), (1, 257, 257, 2, 2, 80), (2, 300, 300, 2, 1, 40), (1, 200, 200, 2, 2, 8),
          (1, 520, 520, 6, 2, 128), (1, 777, 777, 2, 2, 64), (1, 5, 1500, 4, 2, 64)]


@pytest.mark.parametrize("B,Tq,Tk,H,Hk,N", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_against_the_definition(lib, B, Tq, Tk, H, Hk, N, dtype, causal):
    print(f"\n{B} {Tq} {Tk} {H} {Hk} {N} {dtype} {causal}", flush=True)
    check(*inputs(B, Tq, Tk, H, Hk, N, DT[dtype]), causal=causal)


HOW = {"cap": dict(cap=2.0), "bias": dict(bias=True), "cap and bias": dict(cap=5.0, bias=True), "wide bias": dict(bias=True, causal=False), "prefix": dict(prefix=True),
       "prefix and bias": dict(prefix=True, bias=True), "two documents": dict(doc="two"), "many documents": dict(doc="many"), "padding": dict(doc="padded"),
       "single tokens": dict(doc="one"), "ids that come back": dict(doc="back"), "wide documents": dict(doc="padded", causal=False),
       "all": dict(doc="padded", prefix=True, cap=3.0, bias=True)}


@pytest.mark.parametrize("how", list(HOW))
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,N,dtype", [(2, 90, 90, 2, 1, 64, "bf16"), (3, 200, 333, 4, 2, 128, "fp16"), (2, 400, 400, 2, 2, 64, "bf16"), (2, 1, 150, 2, 1, 128, "bf16")])
def test_masks_caps_and_biases(lib, how, B, Tq, Tk, H, Hk, N, dtype):
    print(f"\n{how} {B} {Tq} {Tk} {H} {Hk} {N} {dtype}", flush=True)
    o = dict(HOW[how])
    if o.pop("bias", False):
        o["slopes"] = torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)
    if "doc" in o:
        o["doc"] = doc_ids(B, Tk, o["doc"], seed=Tk).to(DEV)
    if o.pop("prefix", False):
        o["prefix"] = torch.tensor([Tk // 3, Tk + 5, 0][:B], dtype=torch.int32, device=DEV)
    check(*inputs(B, Tq, Tk, H, Hk, N, DT[dtype], seed=7), **o)


@pytest.mark.parametrize("how", ["none", "cap", "bias", "wide bias", "all"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,N", [(4, 300, 300, 32, 32, 128), (2, 300, 411, 64, 16, 128), (4, 260, 260, 32, 32, 64), (2, 129, 129, 12, 2, 64)])
def test_many_heads(lib, how, B, Tq, Tk, H, Hk, N):
    """Workgroups enough for the large ones of heads of 128; heads in one group and in several."""
    q, k, v, dy = inputs(B, Tq, Tk, H, Hk, N, torch.bfloat16, seed=71)
    how = dict(HOW.get(how, {}))
    if how.pop("bias", False):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1) / H).to(DEV)
    if how.pop("prefix", False):
        how["prefix"] = torch.tensor([Tk // 3, 5, 0, Tk + 9][:B], dtype=torch.int32, device=DEV)
    if "doc" in how:
        how["doc"] = doc_ids(B, Tk, how["doc"], seed=3).to(DEV)
    check(q, k, v, dy, **how)


@pytest.mark.parametrize("how", ["many documents", "padding", "ids that come back", "wide documents", "all"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,N,dtype", [(3, 520, 600, 64, 16, 128, "bf16"), (4, 390, 390, 40, 40, 64, "fp16"), (4, 450, 450, 33, 11, 64, "bf16")])
def test_more_blocks_of_documents_than_run_at_once(lib, how, B, Tq, Tk, H, Hk, N, dtype):
    """Blocks of queries and of keys in the order of their work."""
    o = dict(HOW[how])
    if o.pop("bias", False):
        o["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1) / H).to(DEV)
    if o.pop("prefix", False):
        o["prefix"] = torch.tensor([Tk // 3, 5, 0, Tk + 9][:B], dtype=torch.int32, device=DEV)
    o["doc"] = doc_ids(B, Tk, o["doc"], seed=5).to(DEV)
    check(*inputs(B, Tq, Tk, H, Hk, N, DT[dtype], seed=81), **o)


def test_gradients_that_come_as_views_from_anywhere(lib):
    q, k, v, dy = inputs(1, 70, 70, 2, 1, 64, torch.bfloat16, seed=75)
    odd = torch.zeros(dy.numel() + 3, device=DEV, dtype=dy.dtype)[3:].view_as(dy).copy_(dy)
    t = [z.requires_grad_(True) for z in (q, k, v)]
    y = A.RUN_CUDA(*t)
    got, want = (torch.autograd.grad(y, t, d, retain_graph=True) for d in (odd, dy))
    assert odd.data_ptr() % 16 != 0 and all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_scores(lib, dtype):
    """Scores in the hundreds, of either sign: nothing overflows, and rows that are one key's alone."""
    q, k, v, dy = inputs(1, 150, 150, 2, 2, 64, DT[dtype], seed=3, scale=8.0)
    check(q, k, v, dy, scale=1.0)
    check(q, k, v, dy, scale=1.0, cap=30.0)
    check(q, -k.abs(), v, dy, scale=1.0)


def test_views_of_one_projection(lib):
    B, T, H, Hk, N = 2, 140, 4, 2, 64
    x = randn(B, T, (H + 2 * Hk) * N, seed=5).to(torch.bfloat16).to(DEV)
    q, k, v = (z.unflatten(2, (-1, N)) for z in x.split([H * N, Hk * N, Hk * N], 2))
    dy = randn(B, T, H, N, seed=6).to(torch.bfloat16).to(DEV)
    check(q, k, v, dy)
    heads_first = [z.transpose(1, 2).contiguous().transpose(1, 2) for z in (q, k, v)]
    check(*heads_first, dy)
    y = A.RUN_CUDA(q, k, v)
    assert torch.equal(y, A.RUN_CUDA(*heads_first)) and torch.equal(y, A.RUN_CUDA(*(z.contiguous() for z in (q, k, v))))
    one = x[:, :, :N].unsqueeze(2).expand(B, T, H, N)                # a broadcast query: its gradient is the sum over the heads
    t = [z.detach().requires_grad_(True) for z in (x[:, :, :N].contiguous(), k, v)]
    y = A.RUN_CUDA(t[0].unsqueeze(2).expand(B, T, H, N), t[1], t[2])
    got = torch.autograd.grad([y], t, [dy])
    t2 = [z.detach().contiguous().requires_grad_(True) for z in (one, k, v)]
    want = torch.autograd.grad([A.RUN_CUDA(*t2)], t2, [dy])
    assert torch.equal(got[0], want[0].sum(2)) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_padding_of_any_value_reaches_nothing(lib, value):
    B, T, H, Hk, N = 2, 190, 2, 1, 64
    q, k, v, dy = inputs(B, T, T, H, Hk, N, torch.bfloat16, seed=11)
    doc = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    doc[0, 150:] = -1
    doc[1, :20] = -1
    doc[1, 77:99] = -2
    clean = [z.masked_fill((doc < 0)[:, :, None, None], 0.0) for z in (q, k, v, dy)]
    dirty = [z.masked_fill((doc < 0)[:, :, None, None], value) for z in (q, k, v, dy)]
    for causal in (True, False):
        results = []
        for z in (clean, dirty):
            t = [a.detach().requires_grad_(True) for a in z[:3]]
            y = A.RUN_CUDA(*t, doc=doc, causal=causal)
            results.append([y.detach()] + list(torch.autograd.grad([y], t, [z[3]])))
        for n, a, b in zip(["y", "dq", "dk", "dv"], *results):
            assert torch.equal(a, b), n
            assert not a[doc < 0].any(), n


def test_the_same_bits_every_time_and_a_rows_own(lib):
    """Each row of a batch is what it is alone."""
    q, k, v, dy = inputs(3, 333, 333, 4, 2, 64, torch.bfloat16, seed=13)

    def once(q, k, v, dy):
        t = [z.detach().requires_grad_(True) for z in (q, k, v)]
        y = A.RUN_CUDA(*t, cap=20.0)
        return [y.detach()] + list(torch.autograd.grad([y], t, [dy]))
    want = once(q, k, v, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, once(q, k, v, dy)))
    for b in range(3):
        assert all(torch.equal(a[b:b + 1], c) for a, c in zip(want, once(*(z[b:b + 1] for z in (q, k, v, dy)))))


def test_captured_and_replayed(lib):
    q, k, v, dy = inputs(2, 310, 310, 4, 2, 128, torch.bfloat16, seed=17)
    doc = doc_ids(2, 310, "two", seed=1).to(DEV)
    t = [z.detach().clone().requires_grad_(True) for z in (q, k, v)]

    def once():
        y = A.RUN_CUDA(*t, doc=doc)
        return [y.detach()] + list(torch.autograd.grad([y], t, [dy]))
    (g1, o1), (g2, o2) = graph_of(once), graph_of(once)
    for i in range(4):
        with torch.no_grad():
            for j, z in enumerate(t):
                z.copy_(randn(*z.shape, seed=50 + 10 * i + j).to(z.dtype))
            doc.copy_(doc_ids(2, 310, "padded" if i % 2 else "two", seed=i))
        want = [z.clone() for z in once()]
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for o in (o1, o2):
            assert all(torch.equal(a, b) for a, b in zip(want, o)), i


def test_two_streams_at_once(lib):
    cases = [inputs(2, 600, 600, 4, 4, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [A.RUN_CUDA(*c[:3]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(A.RUN_CUDA(*c[:3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_long_keys_and_tensors_beyond_2_31_elements(lib):
    """A few queries of the end of a long text, of which the last part has a document of its own; the heads lie far apart."""
    Tk, N = 70001, 64
    k = torch.zeros(1, Tk, 1, N, device=DEV, dtype=torch.bfloat16)
    k[:] = randn(Tk, 1, N, seed=1).to(DEV)
    v = randn(1, Tk, 1, N, seed=2).to(torch.bfloat16).to(DEV)
    q = randn(1, 3, 2, N, seed=3).to(torch.bfloat16).to(DEV)
    doc = torch.zeros(1, Tk, dtype=torch.int32, device=DEV)
    dy = randn(1, 3, 2, N, seed=4).to(torch.bfloat16).to(DEV)
    check(q, k, v, dy)
    doc[:, 69000:] = 1
    check(q, k, v, dy, doc=doc)
    big = torch.empty(2, Tk, 16 * 1024, device=DEV, dtype=torch.bfloat16)
    assert big.numel() > 1 << 31
    K, V = big[..., :N].unsqueeze(2), big[..., -N:].unsqueeze(2)
    K.copy_(k.expand(2, -1, -1, -1))
    V.copy_(v.expand(2, -1, -1, -1))
    got = A.RUN_CUDA(q.expand(2, -1, -1, -1).contiguous(), K, V)
    want = A.RUN_CUDA(q, k, v)
    assert torch.equal(got[:1], want) and torch.equal(got[1:], want)


def far_rows(z, store, at):
    """z [1,T,H,N] as a view of `store` [T,step], from column `at` on."""
    view = store[:, at:at + z.shape[2] * z.shape[3]].unflatten(1, z.shape[2:])[None]
    view.copy_(z)
    return view


def passes(q, k, v, dy, **how):
    t = [z.detach().requires_grad_(True) for z in (q, k, v)]
    y = A.RUN_CUDA(*t, **how)
    return [y.detach()] + list(torch.autograd.grad([y], t, [dy]))


@pytest.mark.parametrize("Tq,Tk,step,H,Hk,N,dtype", [(257, 257, 1 << 23, 4, 2, 40, "bf16"), (257, 257, 1 << 23, 2, 2, 128, "fp16"), (70, 131100, 16384, 4, 2, 64, "bf16"),
                                                     (3, 350000, 6144, 2, 1, 96, "fp16")])
def test_rows_that_span_more_than_4_gib(lib, Tq, Tk, step, H, Hk, N, dtype):
    """Queries, keys and values a long way apart in one tensor, in which NaN stands between them: what the same rows side by side give."""
    q, k, v, dy = inputs(1, Tq, Tk, H, Hk, N, DT[dtype], seed=21)
    store = torch.full((Tk, step), float("nan"), device=DEV, dtype=DT[dtype])
    assert store.numel() * 2 >= 1 << 32
    far = [far_rows(z, store[Tk - z.shape[1]:], at) for z, at in ((q, 0), (k, 1024), (v, 2048))]
    for n, a, b in zip(["y", "dq", "dk", "dv"], passes(*far, dy), passes(q, k, v, dy)):
        assert torch.equal(a, b), n


def test_padding_in_rows_that_span_more_than_2_gib(lib):
    Tq, Tk, step, H, Hk, N = 70, 70001, 16384, 4, 2, 96
    q, k, v, dy = inputs(1, Tq, Tk, H, Hk, N, torch.bfloat16, seed=25)
    doc = torch.zeros(1, Tk, dtype=torch.int32, device=DEV)
    doc[0, 100:190], doc[0, 50000:50007], doc[0, -9:-5] = -1, -2, -1
    none = (doc < 0)[:, :, None, None]
    q, k, v, dy = (z.masked_fill(none[:, -z.shape[1]:], 0.0) for z in (q, k, v, dy))
    store = torch.full((Tk, step), float("nan"), device=DEV, dtype=torch.bfloat16)
    assert store.numel() * 2 > 1 << 31
    far = [far_rows(z.masked_fill(none[:, -z.shape[1]:], float("nan")), store[Tk - z.shape[1]:], at) for z, at in ((q, 0), (k, 1024), (v, 2048))]
    for n, a, b in zip(["y", "dq", "dk", "dv"], passes(*far, dy.masked_fill(none[:, -Tq:], float("nan")), doc=doc), passes(q, k, v, dy, doc=doc)):
        assert torch.equal(a, b), n


@pytest.mark.parametrize("doc", [None, "two", "padded"])
def test_prefixes_below_zero_are_none(lib, doc):
    B, T, H, Hk, N = 3, 200, 4, 2, 64
    q, k, v, dy = inputs(B, T, T, H, Hk, N, torch.bfloat16, seed=121)
    how = {} if doc is None else dict(doc=doc_ids(B, T, doc, seed=6).to(DEV))
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    want = passes(q, k, v, dy, prefix=at(0, 0, 0), **how)
    for low in (at(-1, -64, -65), at(-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 63)):
        for n, a, b in zip(["y", "dq", "dk", "dv"], passes(q, k, v, dy, prefix=low, **how), want):
            assert torch.equal(a, b), n


@pytest.mark.parametrize("Tq,Tk,H,Hk,N,how", [(200, 4096, 2, 1, 64, {}), (64, 16384, 2, 2, 64, {}), (130, 4096, 4, 1, 128, {}), (64, 16384, 2, 1, 96, dict(cap=30.0)), (4096, 4096, 1, 1, 64, {})])
@pytest.mark.parametrize("up", [1e-2, 1e-3])
def test_small_gradients_over_many_keys(lib, Tq, Tk, H, Hk, N, how, up):
    """fp16: gradients of scores far below the type's normal numbers, for gradients of y as they are in training."""
    q, k, v, dy = inputs(1, Tq, Tk, H, Hk, N, torch.float16, seed=101)
    check(q, k, v, (dy.float() * up).half(), **how)


@pytest.mark.parametrize("Tq,Tk,H,Hk,N", [(300, 300, 2, 1, 64), (150, 2000, 4, 2, 128), (64, 4096, 2, 2, 64)])
def test_large_gradients(lib, Tq, Tk, H, Hk, N):
    """fp16: gradients of scores beyond the type's largest number, where those of q, k and v are not.  (The first shape's reach 1.2e5 in 64 bits: from 65520 on, half a step
    above 65504, a value rounds to infinity in fp16.)"""
    q, k, v, dy = inputs(1, Tq, Tk, H, Hk, N, torch.float16, seed=105)
    got = passes(q, k, v * 4, dy * 1e4)
    want = O.attention(q, k, v * 4, dy=dy * 1e4)
    for n, z in zip(["y", "dq", "dk", "dv"], got):
        value, bound = want[n]
        above, below = value.abs() - bound > 65520, value.abs() + bound < 65520
        assert torch.equal(z[above].float(), torch.sign(value[above]).float() * torch.inf), n
        within(n, z[below], (value[below], bound[below]))
        assert below.float().mean() > 0.99


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 65504.0])
def test_padding_of_any_value_reaches_nothing_in_fp16(lib, value):
    B, T, H, Hk, N = 2, 400, 4, 2, 128
    q, k, v, dy = inputs(B, T, T, H, Hk, N, torch.float16, seed=109)
    doc = doc_ids(B, T, "padded", seed=3).to(DEV)
    doc[1, 60:], doc[1, 200:] = 4, -1
    results = []
    for x in (0.0, value):
        t = [z.masked_fill((doc < 0)[:, :, None, None], x).requires_grad_(True) for z in (q, k, v)]
        y = A.RUN_CUDA(*t, doc=doc)
        results.append([y.detach()] + list(torch.autograd.grad([y], t, [(dy * 1e-3).masked_fill((doc < 0)[:, :, None, None], x)])))
    for n, a, b in zip(["y", "dq", "dk", "dv"], *results):
        assert torch.equal(a, b), n


def test_fp16_rows_on_their_own_and_in_graphs(lib):
    """Gradients of different sizes in the elements of a batch; the same bits every time, in a graph too."""
    q, k, v, dy = inputs(3, 333, 333, 4, 2, 64, torch.float16, seed=113)
    dy = dy * torch.tensor([1.0, 1e-4, 300.0], device=DEV).half().view(3, 1, 1, 1)
    t = [z.detach().clone().requires_grad_(True) for z in (q, k, v)]

    def once(q, k, v, dy):
        y = A.RUN_CUDA(q, k, v)
        return [y.detach()] + list(torch.autograd.grad([y], [q, k, v], [dy]))
    graph, out = graph_of(lambda: once(*t, dy))
    for i in range(4):
        with torch.no_grad():
            dy.mul_(0.5), t[2].copy_(randn(*v.shape, seed=120 + i, scale=2.0 ** i).half())
        want = [z.clone() for z in once(*t, dy)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), i
    for b in range(3):
        alone = [z[b:b + 1].detach().requires_grad_(True) for z in t]
        assert all(torch.equal(a[b:b + 1], c) for a, c in zip(want, once(*alone, dy[b:b + 1])))


@pytest.mark.parametrize("how", [dict(causal=False), dict(prefix=True), dict(cap=3.0, causal=False)])
def test_slopes_with_the_smallest_scale(lib, how):
    """Scores of nothing but the bias, on both sides of a query; a smaller scale is refused where there are slopes."""
    q, k, v, dy = inputs(2, 150, 150, 4, 2, 64, torch.bfloat16, seed=131)
    slopes = torch.exp2(-torch.arange(1.0, 5.0)).to(DEV)
    if "prefix" in how:
        how = dict(prefix=torch.tensor([100, 7], dtype=torch.int32, device=DEV))
    check(q, k, v, dy, slopes=slopes, scale=2.0 ** -60, **how)
    with pytest.raises(AssertionError, match="scale"):
        A.RUN_CUDA(q, k, v, slopes=slopes, scale=2.0 ** -61, **how)
    check(q, k, v, dy, scale=2.0 ** -61, **how)
