"""GPU: the gated delta rule against its 64-bit definition."""
import ctypes

import pytest
import torch

from oracle import delta as O
from rwkv_cuda_amd import _lib, gated_delta as G
from _delta_util import inputs, near
from _gpu_util import DEV
from _mixers_util import DT, doc_ids, graph_of, randn

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "ds0")


def check(t, s0, doc=None, dy=None, dsT=None, scale=None, steps=1.0):
    """Both directions, or without dy and dsT the forward alone."""
    want = O.gated_delta(*t, s0=s0, doc=doc, scale=scale, dy=dy, dsT=dsT)
    grad = dy is not None or dsT is not None
    leaves = [z.detach().requires_grad_(grad) for z in (*t, s0) if z is not None]
    y, sT = G.RUN_CUDA(*leaves[:5], s0=leaves[5] if s0 is not None else None, doc=doc, scale=scale)
    got = dict(y=y, sT=sT)
    if grad:
        out, d = zip(*[(o, g) for o, g in ((y, dy), (sT, dsT)) if g is not None])
        got.update(zip(NAMES, torch.autograd.grad(out, leaves, d)))
    torch.cuda.synchronize()
    for n in got:
        near(n, got[n], want[n], steps)
    return got


@pytest.mark.parametrize("T", [1, 2, 3, 9, 15, 16, 17, 63, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("H,Hk,N,dtype", [(2, 2, 64, "bf16"), (4, 2, 128, "fp16"), (3, 1, 24, "bf16")])
def test_lengths(lib, T, H, Hk, N, dtype):
    print(f"\nT={T} H={H} Hk={Hk} N={N} {dtype}", flush=True)
    t, s0, dy, dsT = inputs(2, T, H, Hk, N, DT[dtype], seed=T)
    check(t, s0, None, dy, dsT)
    check(t, None)


@pytest.mark.parametrize("B,T,H,Hk,N,dtype", [(1, 300, 1, 1, 8, "bf16"), (2, 130, 6, 2, 80, "fp16"), (3, 77, 8, 8, 96, "bf16"), (1, 700, 2, 1, 128, "bf16"), (2, 333, 4, 4, 64, "fp16"), (5, 66, 16, 2, 32, "bf16"),
                                              (1, 70, 36, 36, 64, "bf16"), (9, 65, 40, 8, 112, "fp16"), (2, 64, 5, 5, 40, "fp16")])
def test_heads(lib, B, T, H, Hk, N, dtype):
    print(f"\nB={B} T={T} H={H} Hk={Hk} N={N} {dtype}", flush=True)
    t, s0, dy, dsT = inputs(B, T, H, Hk, N, DT[dtype], seed=N)
    check(t, s0, None, dy, dsT)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hk,N", [(2, 40, 40, 64), (4, 40, 20, 64), (2, 24, 24, 128), (2, 48, 16, 128), (3, 30, 30, 112), (5, 24, 8, 40)])
def test_every_width_of_the_walks(lib, B, H, Hk, N, dtype):
    """Heads for two and for four column tiles a workgroup, some of them beyond the last channel."""
    T = 140
    t, s0, dy, dsT = inputs(B, T, H, Hk, N, DT[dtype], seed=H)
    check(t, s0, doc_ids(B, T, "many", seed=N).to(DEV), dy, dsT)


@pytest.mark.parametrize("kind", ["two", "many", "padded", "one", "back"])
@pytest.mark.parametrize("T,N,dtype", [(7, 64, "bf16"), (150, 64, "fp16"), (200, 128, "bf16"), (64, 40, "fp16")])
def test_documents(lib, kind, T, N, dtype):
    print(f"\n{kind} T={T} N={N} {dtype}", flush=True)
    t, s0, dy, dsT = inputs(3, T, 4, 2, N, DT[dtype], seed=T)
    doc = doc_ids(3, T, kind, seed=T).to(DEV)
    check(t, s0, doc, dy, dsT)
    check(t, None, doc, dy)


@pytest.mark.parametrize("cuts", [[], [1], [300], [320], [384], [511, 513], [63, 700], [704], [767], [100, 101, 102, 400, 640], list(range(1, 768))])
@pytest.mark.parametrize("N,dtype", [(64, "bf16"), (128, "fp16"), (40, "fp16")])
def test_rows_walked_by_two_workgroups(lib, N, dtype, cuts):
    """Twelve chunks: documents that begin nowhere, in the first and last chunk only, at chunks' edges, several in a chunk, everywhere; another row without any, and padding around cuts."""
    T = 768
    t, s0, dy, dsT = inputs(3, T, 4, 2, N, DT[dtype], seed=len(cuts) + N)
    doc = torch.zeros(3, T, dtype=torch.int32)
    for c in cuts:
        doc[0, c:] += 1
    doc[2] = doc[0]
    for c in cuts[:3]:
        doc[2, max(0, c - 5):c] = -1
    doc[2, -70:] = -1
    check(t, s0, doc.to(DEV), dy, dsT)
    check(t, None, doc.to(DEV), dy)


def test_padding_counts_nowhere(lib):
    """NaN and infinities in padding, before, between and behind; rows that are nothing else; dy there too."""
    for N, T, value in ((64, 150, float("nan")), (128, 70, float("inf")), (64, 5, float("nan"))):
        t, s0, dy, dsT = inputs(3, T, 2, 2, N, torch.bfloat16, seed=3)
        doc = doc_ids(3, T, "padded", seed=T).to(DEV)
        bad = doc < 0
        want = check(t, s0, doc, torch.where(bad[:, :, None, None], 0, dy), dsT)
        t2 = [torch.where(bad.view(3, T, *[1] * (z.dim() - 2)), value, z).to(z.dtype) for z in (*t, dy)]
        leaves = [z.requires_grad_(True) for z in (*t2[:5], s0.clone())]
        y, sT = G.RUN_CUDA(*leaves, doc)
        got = [y, sT, *torch.autograd.grad([y, sT], leaves, [t2[5], dsT])]
        for n, g in zip(("y", "sT") + NAMES, got):
            assert torch.equal(g, want[n]), n
            if n not in ("sT", "ds0"):
                assert not g[bad].any(), n


@pytest.mark.parametrize("T", [6, 140])
def test_gates_at_their_ends(lib, T):
    """Decays of nothing, of everything and beyond; beta of 0, 1 and between 1 and 2; the same key over and over."""
    t, s0, dy, dsT = inputs(2, T, 3, 3, 64, torch.bfloat16, seed=5)
    q, k, v, g, beta = t
    g[:, ::5], g[:, 1::7], g[:, 3::11] = 0.0, -120.0, -float("inf")
    g[0, T // 2:] = 0.0
    beta[:, ::4], beta[:, 1::4] = 1.0, 0.0
    beta[1, :, 2] = 1.5
    k[0, :, 1] = k[0, :1, 1]
    got = check(t, s0, None, dy, dsT, steps=2.0)                 # (sums of a hundred equal terms: errors of one sign)
    assert all(torch.isfinite(z).all() for z in got.values()) and not got["dg"][g < -104].any()


def test_strong_decays_beside_weak_ones(lib):
    """Sums of log decays in the thousands, differences of which count to their last bits."""
    t, s0, dy, dsT = inputs(1, 200, 2, 2, 64, torch.bfloat16, seed=6)
    t[3][:, ::2] = -90.0
    t[3][:, 1::2] = -0.01
    t[3][:, 100:] = -0.003
    check(t, s0, None, dy, dsT)


@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** 20])
def test_sizes_far_from_one(lib, size):
    """Values, states and gradients of any size: bf16 has fp32's range."""
    t, s0, dy, dsT = inputs(2, 100, 2, 2, 64, torch.bfloat16, seed=7)
    t[2] = (t[2].float() * size).to(torch.bfloat16)
    check(t, s0 * size, None, (dy.float() * size).to(torch.bfloat16), dsT * size)


def test_small_gradients_in_fp16(lib):
    """Gradients near the end of fp16 (its least step is 2^-24): as exact as their type."""
    t, s0, dy, dsT = inputs(2, 100, 2, 2, 64, torch.float16, seed=8)
    check(t, s0, None, (dy.float() * 2.0 ** -10).half(), dsT * 2.0 ** -10)
    check([t[0], t[1], t[2] * 64, t[3], t[4]], s0 * 64, None, (dy.float() * 8).half(), dsT)


def test_only_one_of_the_outputs_has_a_gradient(lib):
    t, s0, dy, dsT = inputs(2, 90, 2, 2, 64, torch.bfloat16, seed=9)
    check(t, s0, None, dy, None)
    check(t, s0, None, None, dsT)
    leaf = t[2].detach().requires_grad_(True)
    y, _ = G.RUN_CUDA(t[0], t[1], leaf, t[3], t[4])
    y.float().sum().backward()                                   # an upstream gradient with strides of zero
    assert leaf.grad.shape == leaf.shape


def test_views_and_broadcasts(lib):
    """Views of one projection, tokens first in memory, gates at odd offsets; keys and values that all heads or tokens share."""
    B, T, H, Hk, N = 2, 100, 4, 2, 64
    t, s0, dy, dsT = inputs(B, T, H, Hk, N, torch.bfloat16, seed=10)
    want = G.RUN_CUDA(*t, s0)
    both = torch.cat([z.flatten(2) for z in t[:3]], 2)
    q, k, v = (z.unflatten(2, (-1, N)) for z in both.split([Hk * N, Hk * N, H * N], 2))
    gates = torch.cat([t[3], t[4], t[3]], 2)
    views = [q, k, v, gates[..., 1:1 + H], gates[..., H:2 * H]]
    assert all(torch.equal(a, b) for a, b in zip(G.RUN_CUDA(q, k, v, gates[..., :H], gates[..., H:2 * H], s0), want))
    check(views, s0, None, dy, dsT)
    turned = [z.transpose(0, 1).contiguous().transpose(0, 1) for z in t]
    assert all(torch.equal(a, b) for a, b in zip(G.RUN_CUDA(*turned, s0), want))
    one = [t[0], t[1][:, :, :1].expand(B, T, Hk, N), t[2][:, :1].expand(B, T, H, N), t[3], t[4]]
    small = [one[0], t[1][:, :, :1].detach().requires_grad_(True), t[2][:, :1].detach().requires_grad_(True)]
    y, _ = G.RUN_CUDA(one[0], small[1].expand(B, T, Hk, N), small[2].expand(B, T, H, N), t[3], t[4])
    dk, dv = torch.autograd.grad(y, small[1:], dy)
    ref = O.gated_delta(*one, dy=dy)
    assert dk.shape == small[1].shape and dv.shape == small[2].shape
    # (torch adds the heads' and tokens' gradients, rounded to 8 bits, in 32 bits and rounds once more)
    assert float((dv.double() - ref["dv"].sum(1, keepdim=True)).norm() / ref["dv"].sum(1).norm()) < 2.0 ** -6
    assert float((dk.double() - ref["dk"].sum(2, keepdim=True)).norm() / ref["dk"].sum(2).norm()) < 2.0 ** -6


def test_two_calls_pass_the_state_on(lib):
    t, s0, _, _ = inputs(2, 300, 4, 2, 128, torch.bfloat16, seed=11)
    want = O.gated_delta(*t, s0=s0)
    for cut in (1, 5, 64, 130, 299):
        y0, s = G.RUN_CUDA(*(z[:, :cut] for z in t), s0)
        y1, sT = G.RUN_CUDA(*(z[:, cut:] for z in t), s)
        near("y", torch.cat([y0, y1], 1), want["y"])
        near("sT", sT, want["sT"])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,Hk,N", [(1, 1, 1, 8), (3, 6, 2, 80), (32, 16, 16, 64), (5, 8, 4, 128)])
def test_step(lib, dtype, B, H, Hk, N):
    """A token at a time gives what whole sequences do, in place and into other memory."""
    T = 5
    t, s0, _, _ = inputs(B, T, H, Hk, N, DT[dtype], seed=12)
    want = O.gated_delta(*t, s0=s0)
    s, keep = s0.clone(), s0.clone()
    other = torch.empty_like(s)
    ys = []
    for i in range(T):
        now = [z[:, i] for z in t]
        ys.append(G.STEP(*now, keep, out=other))
        version = s._version
        assert torch.equal(ys[-1], G.STEP(*now, s)) and torch.equal(s, other) and s._version > version
        keep, other = other, keep
    near("y", torch.stack(ys, 1), want["y"])
    near("s", s, want["sT"])


def test_the_same_bits_every_time_and_alone(lib):
    t, s0, dy, dsT = inputs(3, 210, 4, 2, 64, torch.bfloat16, seed=13)

    def once(t, s0, dy, dsT):
        leaves = [z.detach().requires_grad_(True) for z in (*t, s0)]
        y, sT = G.RUN_CUDA(*leaves)
        return [y.detach(), sT.detach(), *torch.autograd.grad([y, sT], leaves, [dy, dsT])]
    want = once(t, s0, dy, dsT)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, once(t, s0, dy, dsT)))


def test_captured_and_replayed(lib):
    """Forward and backward in a graph, replayed on changing inputs between eager calls; two graphs of the same leaves; the single token."""
    t, s0, dy, dsT = inputs(2, 150, 4, 2, 64, torch.bfloat16, seed=14)
    leaves = [z.detach().clone().requires_grad_(True) for z in (*t, s0)]

    def once():
        y, sT = G.RUN_CUDA(*leaves)
        return [y.detach(), sT.detach(), *torch.autograd.grad([y, sT], leaves, [dy, dsT])]
    (g1, o1), (g2, o2) = graph_of(once), graph_of(once)
    now, s = [z[:, 0].clone() for z in t], s0.clone()
    out = torch.empty_like(s)
    g3, o3 = graph_of(lambda: G.STEP(*now, s, out=out))
    for i in range(4):
        with torch.no_grad():
            leaves[2].copy_(randn(*t[2].shape, seed=100 + i).to(t[2].dtype))
            now[2].copy_(leaves[2][:, 1])
        want = [z.clone() for z in once()]
        step = G.STEP(*now, s, out=out).clone()
        after = out.clone()
        out.zero_()
        for g in (g1, g2, g3):
            g.replay()
        torch.cuda.synchronize()
        for o in (o1, o2):
            assert all(torch.equal(a, b) for a, b in zip(want, o)), i
        assert torch.equal(step, o3) and torch.equal(after, out)


def test_two_streams_at_once(lib):
    cases = [inputs(2, 200, 4, 4, 64, torch.bfloat16, seed=s)[0] for s in (1, 2)]
    want = [G.RUN_CUDA(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(G.RUN_CUDA(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for m, n in zip(want, got) for a, b in zip(m, n))


def test_tokens_far_apart_and_long_rows(lib):
    """[T,B,...] in memory, offsets of a chunk beyond 32 bits; only some rows are looked at."""
    T, B, H, N = 70, 32768, 16, 64
    small = inputs(1, T, H, H, N, torch.bfloat16, seed=15)[0]
    far = [z.transpose(0, 1).expand(T, B, *z.shape[2:]) for z in small]
    v = far[2].contiguous().transpose(0, 1)
    k = far[1].contiguous().transpose(0, 1)
    assert v.stride(1) * 2 * (T - 1) > 1 << 32 and v.numel() > 1 << 31
    one = lambda z: z.transpose(0, 1)
    y, sT = G.RUN_CUDA(one(far[0]), k, v, one(far[3]).contiguous(), one(far[4]).contiguous())
    want = G.RUN_CUDA(*small)
    assert all(torch.equal(y[b], want[0][0]) and torch.equal(sT[b], want[1][0]) for b in (0, 1, 1000, B - 1))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N,kind", [(64, None), (128, "many"), (24, "padded"), (80, "one")])
def test_what_memory_held_before_counts_nowhere(lib, N, kind, dtype):
    """The same bits whatever the outputs' and the workspaces' memory held: zeros, NaN, large numbers; and again, twenty times."""
    t, s0, dy, dsT = inputs(3, 200, 4, 2, N, DT[dtype], seed=N)
    doc = None if kind is None else doc_ids(3, 200, kind, seed=N).to(DEV)
    first = None
    for value in [0.0, float("nan"), 1e4] + 20 * [None]:
        if value is not None:
            held = [torch.full((n,), value, device=DEV) for n in (1 << 8, 1 << 12, 1 << 16, 1 << 18, 1 << 20) for _ in range(12)]
            torch.cuda.synchronize()
            del held
        leaves = [z.detach().requires_grad_(True) for z in (*t, s0)]
        y, sT = G.RUN_CUDA(*leaves[:5], s0=leaves[5], doc=doc)
        got = [y.detach(), sT.detach(), *torch.autograd.grad((y, sT), leaves, (dy, dsT))]
        first = got if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(first, got)), value


def rows_of(lengths, T, pad=None):
    """[1,T] of documents of these lengths, `pad` (begin, end) of it padding."""
    doc = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)])
    assert doc.numel() == T
    if pad:
        doc[pad[0]:pad[1]] = -1
    return doc[None]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gate_gradients_of_documents_beside_each_other(lib, dtype):
    """What a document's gradients are does not depend on the others of its 64 tokens: none where it has no dy, however large theirs are, and as exact as alone where they are a millionth."""
    lengths = [20, 12, 17, 15, 40, 30]
    T = sum(lengths)
    doc = rows_of(lengths, T).to(DEV)
    t, _, dy, _ = inputs(1, T, 3, 3, 64, DT[dtype], seed=17)
    t[3][:, 25] = -110.0                                         # (a decay of nothing is where a document might begin)
    dy[:, 32:49] = 0
    dy[:, 64:104] *= 2.0 ** -10
    dy[:, :20] *= 2.0 ** 6
    leaves = [z.requires_grad_(True) for z in t]
    y, _ = G.RUN_CUDA(*leaves, doc=doc)
    got = dict(zip(NAMES, torch.autograd.grad(y, leaves, dy)))
    want = O.gated_delta(*t, doc=doc, dy=dy)
    at = 0
    for n in lengths:
        print(f"\n{n} tokens from {at} on", flush=True)
        for name in got:
            if not dy[:, at:at + n].any():
                assert not got[name][:, at:at + n].any(), name
            near(name, got[name][:, at:at + n], want[name][:, at:at + n], steps=2.0)
        at += n


@pytest.mark.parametrize("H,N,dtype", [(2, 64, "bf16"), (4, 128, "fp16"), (3, 40, "bf16")])
@pytest.mark.parametrize("lengths,pad", [([2, 2], None), ([4, 5, 3], (7, 9)), ([64, 64, 64], None), ([10, 54, 36, 50], (140, 150)), ([30, 9, 9, 9, 73], None), ([300, 100, 240, 128], (380, 410))])
def test_what_is_no_number_stays_in_its_document(lib, lengths, pad, H, N, dtype):
    """An infinity, a NaN or a state that overflows in one document, whatever it comes from: the others' outputs and gradients are those without it, padding has none."""
    T, dt = sum(lengths), DT[dtype]
    doc = rows_of(lengths, T, pad).to(DEV)
    t, s0, dy, dsT = inputs(1, T, H, 1 if H == 3 else 2, N, dt, seed=T)
    want = O.gated_delta(*t, s0=s0, doc=doc, dy=dy, dsT=dsT)
    begins = [sum(lengths[:i]) for i in range(len(lengths))]
    for bad in range(len(lengths)):
        real = [i for i in range(begins[bad], begins[bad] + lengths[bad]) if int(doc[0, i]) >= 0]
        at, last = real[len(real) // 2], real[-1]
        for what in ("q", "k", "v", "g", "grows", "beta", "dy", "s0", "dsT"):
            if (what == "s0" and bad > 0) or (what == "dsT" and bad + 1 < len(lengths)) or (what == "grows" and len(real) < 12):
                continue
            print(f"\n{lengths} H={H} N={N} {dtype}: document {bad}, {what}", flush=True)
            x = dict(zip(("q", "k", "v", "g", "beta", "s0", "dy", "dsT"), [z.clone() for z in (*t, s0, dy, dsT)]))
            if what == "grows":
                x["k"][0, real[0]:last + 1] *= 1e15 if dt == torch.bfloat16 else 1e3
            elif what in ("s0", "dsT"):
                x[what][0, 0, 1, 3] = float("inf")
            elif what in ("g", "beta"):
                x[what][0, at, 0] = float("nan") if what == "beta" else float("inf")
            else:
                x[what][0, at, 0, 1] = float("nan") if what == "k" else float("inf")
            leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "g", "beta", "s0")]
            y, sT = G.RUN_CUDA(*leaves, doc)
            got = dict(zip(("y", "sT") + NAMES, (y, sT, *torch.autograd.grad([y, sT], leaves, [x["dy"], x["dsT"]]))))
            y0, s1 = G.RUN_CUDA(*[z.detach() for z in leaves], doc)      # (another way for a few tokens)
            torch.cuda.synchronize()
            others = torch.zeros(1, T, dtype=torch.bool, device=DEV)
            others[0, [i for i in range(T) if int(doc[0, i]) >= 0 and not begins[bad] <= i < begins[bad] + lengths[bad]]] = True
            for n in got:
                if n in ("sT", "ds0"):
                    if bad != (len(lengths) - 1 if n == "sT" else 0):
                        near(n, got[n], want[n])
                else:
                    near(n, got[n][others], want[n][others])
                    assert not got[n][doc < 0].any(), n
            near("y", y0[others], want["y"][others])
            assert not y0[doc < 0].any()
            if bad + 1 < len(lengths):
                near("sT", s1, want["sT"])
            if what not in ("q", "dy", "dsT"):                   # ... and is seen there
                assert not torch.isfinite(y[0, last]).all() and not torch.isfinite(y0[0, last]).all()
            assert not all(torch.isfinite(got[n][0, begins[bad]:last + 1]).all() for n in ("y", "dq", "dk", "dv", "dg", "dbeta"))


@pytest.mark.parametrize("T,at", [(4, 2), (60, 30), (200, 64), (200, 101)])
@pytest.mark.parametrize("N,dtype", [(64, "fp16"), (128, "bf16")])
def test_a_decay_of_nothing_lets_no_infinity_through(lib, T, at, N, dtype):
    t, s0, dy, dsT = inputs(2, T, 2, 2, N, DT[dtype], seed=19)
    t[3][:, at] = -float("inf")
    want = O.gated_delta(*t, s0=s0, dy=dy, dsT=dsT)
    for before in (True, False):
        x = [z.clone() for z in (*t, s0, dy, dsT)]
        if before:
            x[2][:, at - 2], x[5][0, 1, 2, 3] = float("inf"), float("nan")
        else:
            x[6][:, at + 1], x[7][0, 1, 2, 3] = -float("inf"), float("nan")
        leaves = [z.requires_grad_(True) for z in x[:6]]
        y, sT = G.RUN_CUDA(*leaves)
        got = dict(zip(("y", "sT") + NAMES, (y, sT, *torch.autograd.grad([y, sT], leaves, x[6:]))))
        rest = slice(at, None) if before else slice(None, at)
        for n in got:
            if n not in ("sT", "ds0"):
                near(n, got[n][:, rest], want[n][:, rest])
        near("sT", sT, want["sT"]) if before else near("ds0", got["ds0"], want["ds0"])


def test_infinities_in_one_value_channel_of_fp16(lib):
    """Value channels do not depend on each other: the others' outputs, states and gradients are those without the infinity."""
    t, s0, dy, dsT = inputs(2, 200, 3, 3, 64, torch.float16, seed=18)
    want = O.gated_delta(*t, s0=s0, dy=dy, dsT=dsT)
    rest = [c for c in range(64) if c != 5]
    for name in ("v", "s0", "dy", "dsT"):
        x = dict(v=t[2].clone(), s0=s0.clone(), dy=dy.clone(), dsT=dsT.clone())
        if name in ("v", "dy"):
            x[name][:, 100, :, 5] = float("inf")
        else:
            x[name][:, :, 7, 5] = -float("inf")
        leaves = [t[0], t[1], x["v"], t[3], t[4], x["s0"]]
        for z in leaves:
            z.requires_grad_(True)
        y, sT = G.RUN_CUDA(*leaves)
        dv, ds0 = torch.autograd.grad([y, sT], [leaves[2], leaves[5]], [x["dy"], x["dsT"]])
        print(f"\n{name}", flush=True)
        near("y", y[..., rest], want["y"][..., rest])
        near("sT", sT[..., rest], want["sT"][..., rest])
        near("dv", dv[..., rest], want["dv"][..., rest])
        near("ds0", ds0[..., rest], want["ds0"][..., rest])
        assert not all(torch.isfinite(z[..., 5]).all() for z in (y, sT, dv, ds0))


@pytest.mark.parametrize("cuts", [[], [300], [384, 500]])
@pytest.mark.parametrize("B,T,H,N,dtype", [(1, 768, 4, 64, "bf16"), (1, 1024, 32, 128, "fp16"), (2, 3, 2, 64, "bf16")])
def test_states_in_place(lib, B, T, H, N, dtype, cuts):
    """By the C ABI, sT in the memory of s0 and ds0 in that of dsT: the bits of separate tensors, also in rows of documents that two workgroups would walk."""
    dt = DT[dtype]
    t, s0, dy, dsT = inputs(B, T, H, H, N, dt, seed=20)
    doc = torch.zeros(B, T, dtype=torch.int32)
    for c in cuts:
        doc[:, c:] += 1
    doc = doc.to(DEV)
    q, k, v, g, beta = t
    wide, gate = (T * H * N, H * N, N), (T * H, H)
    at = lambda z: None if z is None else z.data_ptr()
    res = []
    for place in (False, True):
        a, b = s0.clone(), dsT.clone()
        sT, ds0 = (a, b) if place else (torch.full_like(s0, float("nan")), torch.full_like(s0, float("nan")))
        new = lambda *s: torch.empty(*s, dtype=dt, device=DEV)
        y, d, dgates = new(B, T, H, N), [new(B, T, H, N) for _ in range(3)], [new(B, T, H) for _ in range(2)]
        saved = torch.empty(lib.rwkv_delta_saved_bytes(B, T, H, H, N), dtype=torch.uint8, device=DEV)
        ws = torch.empty(max(16, lib.rwkv_delta_workspace_bytes(B, T, H, H, N, 1)), dtype=torch.uint8, device=DEV)
        args = _lib.DeltaArgs(dtype=0 if dt == torch.bfloat16 else 1, B=B, T=T, H=H, Hk=H, N=N, scale=0.125, q=at(q), k=at(k), v=at(v), g=at(g), beta=at(beta), s0=at(a), doc=at(doc), y=at(y), sT=at(sT),
                              saved=at(saved), saved_bytes=saved.numel(), dy=at(dy), dsT=at(b), dq=at(d[0]), dk=at(d[1]), dv=at(d[2]), dg=at(dgates[0]), dbeta=at(dgates[1]), ds0=at(ds0), workspace=at(ws),
                              workspace_bytes=ws.numel(), **{f"{n}_{s}": x for n in "qkv" for s, x in zip(("sb", "st", "sh"), wide)}, **{f"{n}_{s}": x for n in ("g", "beta") for s, x in zip(("sb", "st"), gate)})
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.rwkv_delta_forward(stream, ctypes.byref(args)) == 0 and lib.rwkv_delta_backward(stream, ctypes.byref(args)) == 0
        torch.cuda.synchronize()
        res.append([y, sT, *d, *dgates, ds0])
    want = O.gated_delta(*t, s0=s0, doc=doc, scale=0.125, dy=dy, dsT=dsT)
    for n, x, z in zip(("y", "sT") + NAMES, *res):
        assert torch.equal(x, z), n
        near(n, z, want[n])


@pytest.mark.parametrize("cuts", [[1], [300, 384], [448], [100, 101, 102, 400, 640], [767]])
@pytest.mark.parametrize("B,H,Hk,N,dtype", [(1, 32, 16, 128, "bf16"), (1, 32, 32, 120, "fp16"), (2, 32, 8, 64, "fp16"), (1, 64, 64, 40, "bf16")])
def test_rows_walked_by_two_workgroups_of_two_column_tiles(lib, B, H, Hk, N, dtype, cuts):
    """As above with as many heads as make workgroups of two tiles the fewest rounds, some of whose channels are behind the last."""
    T = 768
    t, s0, dy, dsT = inputs(B, T, H, Hk, N, DT[dtype], seed=N)
    doc = torch.zeros(B, T, dtype=torch.int32)
    for c in cuts:
        doc[:, c:] += 1
    doc[-1, cuts[0] - 1:cuts[0]] = -1
    check(t, s0, doc.to(DEV), dy, dsT)


@pytest.mark.parametrize("B,T,H,Hk,N,dtype", [(4, 140, 40, 20, 64, "fp16"), (2, 140, 24, 24, 128, "bf16"), (3, 100, 30, 30, 112, "fp16"), (1, 768, 32, 16, 128, "bf16")])
def test_what_is_no_number_in_one_row_and_head(lib, B, T, H, Hk, N, dtype):
    """Walks of two and four column tiles, and by two workgroups: other rows and heads keep their bits, other documents of the row are as without it, twice the same."""
    dt = DT[dtype]
    t, s0, dy, dsT = inputs(B, T, H, Hk, N, dt, seed=21)
    doc = torch.zeros(B, T, dtype=torch.int32)
    doc[:, T // 3:] += 1
    doc[:, T // 2 + 3:] += 1
    doc = doc.to(DEV)

    def once(t, s0, dy, dsT):
        leaves = [z.detach().clone().requires_grad_(True) for z in (*t, s0)]
        y, sT = G.RUN_CUDA(*leaves, doc)
        return dict(zip(("y", "sT") + NAMES, (y.detach(), sT.detach(), *torch.autograd.grad([y, sT], leaves, [dy, dsT]))))
    want = once(t, s0, dy, dsT)
    bad, G_ = H - 1, H // Hk
    v = t[2].clone()
    v[B - 1, T // 3 + 7, bad, N - 1] = float("inf")
    got, again = (once([t[0], t[1], v, *t[3:]], s0, dy, dsT) for _ in range(2))
    of = lambda n, z: z.transpose(1, 2) if n not in ("sT", "ds0") else z          # [B, heads, ...]
    exact = O.gated_delta(*[z[B - 1:] for z in t], s0=s0[B - 1:], doc=doc[B - 1:], dy=dy[B - 1:], dsT=dsT[B - 1:])
    middle = doc[B - 1] == 1
    for n in want:
        a, b = of(n, got[n]), of(n, want[n])
        assert torch.equal(torch.nan_to_num(got[n]), torch.nan_to_num(again[n])), n
        assert torch.equal(a[:B - 1], b[:B - 1]), n
        last = bad // G_ if n in ("dq", "dk") else bad
        assert torch.equal(a[B - 1, :last], b[B - 1, :last]), n
        assert torch.isfinite(got[n][B - 1]).all() if n in ("sT", "ds0") else torch.isfinite(got[n][B - 1, ~middle]).all(), n
        if n in ("sT", "ds0"):
            near(n, got[n][B - 1:], exact[n])
        else:
            near(n, got[n][B - 1, ~middle], exact[n][0, ~middle])
    assert not torch.isfinite(got["y"][B - 1, middle]).all() and not torch.isfinite(got["dk"][B - 1, middle]).all()
