"""GPU: the gated recurrence against its 64-bit definition, with bounds element by element."""
import pytest
import torch

from oracle import mixers as O
from rwkv_cuda_amd import gated_recurrence as G
from _gpu_util import DEV
from _mixers_util import DT, doc_ids, graph_of, randn, within

pytestmark = pytest.mark.gpu


def inputs(B, T, C, dt, gate, seed=0):
    w = randn(B, T, C, seed=seed + 1, shift=2.0) if gate == "sigmoid" else -torch.exp(randn(B, T, C, seed=seed + 1, shift=-3.0))
    return [z.to(dt).to(DEV) for z in (w, randn(B, T, C, seed=seed + 2))] + [randn(B, C, seed=seed + 3).to(DEV), randn(B, T, C, seed=seed + 4).to(dt).to(DEV), randn(B, C, seed=seed + 5).to(DEV)]


def check(w, x, h0, doc, gate, tied, dy, dhT):
    leaves = [z.detach().requires_grad_(True) for z in (w, x)] + ([h0.detach().requires_grad_(True)] if h0 is not None else [])
    y, hT = G.RUN_CUDA(leaves[0], leaves[1], leaves[2] if h0 is not None else None, doc, gate, tied)
    assert y.is_contiguous() and y.dtype == w.dtype and hT.dtype == torch.float32
    up = [(o, g) for o, g in ((y, dy), (hT, dhT)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in up], leaves, [g for _, g in up])
    torch.cuda.synchronize()
    want = O.gated_recurrence(w, x, h0, doc, gate, tied, dy, dhT)
    for n, got in zip(["y", "hT", "dw", "dx", "dh0"], [y, hT] + list(grads)):
        within(n, got, want[n])
    with torch.no_grad():
        y1, hT1 = G.RUN_CUDA(w, x, h0, doc, gate, tied)
    assert torch.equal(y, y1) and torch.equal(hT, hT1)              # what is kept for the backward changes no result


SHAPES = [(1, 1, 1), (2, 1, 64), (3, 2, 7), (2, 15, 33), (1, 16, 64), (2, 17, 130), (2, 63, 100), (1, 255, 66), (2, 512, 64), (1, 513, 96), (3, 600, 37), (1, 1025, 192),
          (2, 1531, 70), (1, 4099, 40)]


@pytest.mark.parametrize("B,T,C", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("gate,tied", [("sigmoid", True), ("log", False)])
def test_against_the_definition(lib, B, T, C, dtype, gate, tied):
    print(f"\n{B} {T} {C} {dtype} {gate} {tied}", flush=True)
    w, x, h0, dy, dhT = inputs(B, T, C, DT[dtype], gate)
    state = (T + C) % 2 == 0
    check(w, x, h0 if state else None, None, gate, tied, dy, dhT if state else None)


@pytest.mark.parametrize("kind", ["two", "many", "padded", "one", "back"])
@pytest.mark.parametrize("B,T,C", [(2, 1, 8), (3, 40, 66), (4, 515, 64), (2, 1300, 72)])
@pytest.mark.parametrize("dtype,gate,tied", [("bf16", "sigmoid", False), ("fp32", "log", True)])
def test_documents_and_padding(lib, kind, B, T, C, dtype, gate, tied):
    print(f"\n{kind} {B} {T} {C} {dtype} {gate} {tied}", flush=True)
    w, x, h0, dy, dhT = inputs(B, T, C, DT[dtype], gate, seed=10)
    check(w, x, h0, doc_ids(B, T, kind, seed=T).to(DEV), gate, tied, dy, dhT)


@pytest.mark.parametrize("B,T,C,kind", [(8, 300, 4096, None), (9, 270, 3649, None), (9, 390, 3650, "padded"), (16, 129, 2048, "many"), (9, 261, 3649, "two")])
@pytest.mark.parametrize("dtype,gate,tied", [("bf16", "sigmoid", True), ("fp16", "log", False), ("fp32", "log", True)])
def test_enough_columns_to_walk_through(lib, B, T, C, kind, dtype, gate, tied):
    """512 columns of 64 channels and more."""
    w, x, h0, dy, dhT = inputs(B, T, C, DT[dtype], gate, seed=90)
    check(w, x, h0, None if kind is None else doc_ids(B, T, kind, seed=T).to(DEV), gate, tied, dy, dhT)


def test_tokens_far_apart(lib):
    """[T,B,C] in memory, a token 2^24 elements from the next: offsets within a tile beyond 32 bits."""
    T, B, C = 66, 4096, 4096
    w, x = (randn(T, 1, C, seed=s).to(torch.bfloat16).to(DEV).expand(T, B, C).contiguous().transpose(0, 1) for s in (1, 2))
    assert w.stride(1) * w.element_size() * (T - 1) > 1 << 31
    y, hT = G.RUN_CUDA(w, x)
    want = G.RUN_CUDA(w[:1].contiguous(), x[:1].contiguous())
    assert all(torch.equal(y[b], want[0][0]) and torch.equal(hT[b], want[1][0]) for b in (0, 1, 2047, 4095))


@pytest.mark.parametrize("gate,tied", [("sigmoid", False), ("log", True)])
def test_only_one_of_the_outputs_has_a_gradient(lib, gate, tied):
    w, x, h0, dy, dhT = inputs(2, 530, 68, torch.float16, gate, seed=20)
    check(w, x, h0, None, gate, tied, dy, None)
    check(w, x, h0, None, gate, tied, None, dhT)
    leaf = w.detach().requires_grad_(True)
    y, hT = G.RUN_CUDA(leaf, x, h0)
    y.sum().backward()                                               # an upstream gradient with strides of zero
    assert leaf.grad.shape == w.shape


@pytest.mark.parametrize("dtype", list(DT))
def test_strided_inputs_and_odd_offsets(lib, dtype):
    """Views of one projection, a transposed batch, and rows that begin at any element."""
    B, T, C = 2, 521, 66
    dt = DT[dtype]
    w, x, h0, dy, dhT = inputs(B, T, C, dt, "sigmoid", seed=30)
    want = G.RUN_CUDA(w, x, h0)
    for make in (lambda z, o: torch.cat([z.new_zeros(B, T, o), z, z.new_zeros(B, T, 5)], 2)[..., o:o + C],
                 lambda z, o: z.transpose(0, 1).contiguous().transpose(0, 1)):
        for offset in (1, 3, 4, 8):
            a, b = make(w, offset), make(x, offset + 1)
            assert not a.is_contiguous()
            got = G.RUN_CUDA(a, b, h0)
            assert all(torch.equal(m, n) for m, n in zip(want, got))
    check(make(w, 1), make(x, 2), h0, None, "sigmoid", True, dy, dhT)
    both = torch.cat([w, x], 2)
    check(both[..., :C], both[..., C:], h0, None, "sigmoid", True, dy, dhT)


@pytest.mark.parametrize("gate", ["sigmoid", "log"])
def test_gates_at_their_ends(lib, gate):
    """A gate of exactly 0 forgets, infinities before it included; one of exactly 1 keeps the state for thousands of steps."""
    B, T, C = 1, 1100, 64
    w, x, h0, dy, dhT = inputs(B, T, C, torch.float32, gate, seed=40)
    w[:, ::3] = -float("inf")
    w[:, 700:] = float("inf") if gate == "sigmoid" else 0.0
    x[:, 700:] *= 0.01
    check(w, x, h0, None, gate, False, None, dhT)
    y = G.RUN_CUDA(w, x, h0, None, gate, False)[0]
    tied = G.RUN_CUDA(w, x, h0, None, gate, True)[0]
    assert torch.isfinite(y).all() and torch.equal(tied[:, 700:], tied[:, 699:700].expand(-1, 400, -1))


def test_what_is_no_number_stays_in_its_channel_and_document(lib):
    B, T, C = 2, 700, 64
    w, x, h0, dy, dhT = inputs(B, T, C, torch.bfloat16, "sigmoid", seed=50)
    doc = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    doc[:, 100:650] = 1
    doc[:, 650:] = -1
    want = G.RUN_CUDA(w, x, h0, doc)[0]
    for z, value in ((x, float("nan")), (w, float("nan")), (x, float("inf"))):
        z2 = z.clone()
        z2[0, 40, 5] = value                                         # in the first document
        z2[:, 660:] = value                                          # padding
        y, hT = G.RUN_CUDA(z2 if z is w else w, z2 if z is x else x, h0, doc)
        bad = ~torch.isfinite(y)
        assert bad[0, 40:100, 5].all() and int(bad.sum()) == 60 and torch.isfinite(hT).all()
        assert torch.equal(y[~bad], want[~bad])


def test_two_calls_pass_the_state_on(lib):
    B, T, C = 2, 900, 72
    w, x, h0, _, _ = inputs(B, T, C, torch.float32, "log", seed=60)
    want = O.gated_recurrence(w, x, h0, None, "log")
    for cut in (1, 512, 777):
        y0, h = G.RUN_CUDA(w[:, :cut], x[:, :cut], h0, gate="log")
        y1, hT = G.RUN_CUDA(w[:, cut:], x[:, cut:], h, gate="log")
        within("y", torch.cat([y0, y1], 1), want["y"])
        within("hT", hT, want["hT"])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("B,C", [(1, 1), (3, 77), (32, 2048)])
def test_step(lib, dtype, B, C):
    """A token at a time gives what whole sequences do, in place and into other memory."""
    T = 5
    w, x, h0, _, _ = inputs(B, T, C, DT[dtype], "sigmoid", seed=70)
    want = O.gated_recurrence(w, x, h0)
    h, keep = h0.clone(), h0.clone()
    other = torch.empty_like(h)
    ys = []
    for t in range(T):
        ys.append(G.STEP(w[:, t], x[:, t], keep, out=other))
        assert torch.equal(ys[-1], G.STEP(w[:, t], x[:, t], h)) and torch.equal(h, other)
        keep, other = other, keep
    within("y", torch.stack(ys, 1), want["y"])
    within("h", h, want["hT"])


def test_the_same_bits_every_time(lib):
    w, x, h0, dy, dhT = inputs(3, 2050, 200, torch.bfloat16, "sigmoid", seed=80)

    def once():
        t = [z.detach().requires_grad_(True) for z in (w, x, h0)]
        y, hT = G.RUN_CUDA(*t)
        return [y.detach(), hT.detach()] + list(torch.autograd.grad([y, hT], t, [dy, dhT]))
    want = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, once()))


def test_captured_and_replayed(lib):
    """Forward and backward in a graph, replayed on changing inputs between eager calls; two graphs of the same leaves."""
    w, x, h0, dy, dhT = inputs(2, 1600, 136, torch.bfloat16, "sigmoid", seed=90)
    t = [z.detach().clone().requires_grad_(True) for z in (w, x, h0)]

    def once():
        y, hT = G.RUN_CUDA(*t)
        return [y.detach(), hT.detach()] + list(torch.autograd.grad([y, hT], t, [dy, dhT]))
    (g1, o1), (g2, o2) = graph_of(once), graph_of(once)
    for i in range(4):
        with torch.no_grad():
            for z, seed in zip(t[:2], (1, 2)):
                z.copy_(randn(*z.shape, seed=100 + 10 * i + seed).to(z.dtype))
        want = [z.clone() for z in once()]
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for o in (o1, o2):
            assert all(torch.equal(a, b) for a, b in zip(want, o)), i


def test_two_streams_at_once(lib):
    cases = [inputs(2, 1700, 264, torch.bfloat16, "sigmoid", seed=s) for s in (1, 2)]
    want = [G.RUN_CUDA(*c[:3]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(G.RUN_CUDA(*c[:3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for m, n in zip(want, got) for a, b in zip(m, n))


def test_a_tensor_of_more_than_2_31_elements(lib):
    """Offsets beyond 32 bits: the last channels of the last rows, against a call on those alone."""
    B, T, C = 3, 96, 1 << 23
    assert B * T * C > 1 << 31
    w = torch.full((1, 1, 1), 2.0, device=DEV, dtype=torch.bfloat16).expand(B, T, C)
    x = torch.zeros(B, T, C, device=DEV, dtype=torch.bfloat16)
    x[:, :, -64:] = randn(B, T, 64, seed=1).to(DEV)
    y, hT = G.RUN_CUDA(w.contiguous(), x)
    want = G.RUN_CUDA(w[:, :, -64:].contiguous(), x[:, :, -64:])
    assert torch.equal(y[:, :, -64:], want[0]) and torch.equal(hT[:, -64:], want[1]) and not y[:, :, :64].any()


@pytest.mark.parametrize("B,T,C", [(1, 129, 64), (2, 1300, 40), (9, 300, 3650), (1, 30, 66)])
@pytest.mark.parametrize("tied", [False, True])
def test_growth_of_nothing_is_nothing(lib, B, T, C, tied):
    """Log gates above 0 over many tokens, on a state of zero and on gradients of zero: their product is beyond fp32, the results are not."""
    w = torch.full((B, T, C), 1.0 if T > 60 else 20.0, device=DEV)
    w[:, T // 2:T // 2 + 8] = 15.0
    x = torch.zeros(B, T, C, device=DEV)
    x[:, -3:] = randn(B, 3, C, seed=1).to(DEV)
    dy = torch.zeros(B, T, C, device=DEV)
    dy[:, :2] = randn(B, 2, C, seed=2).to(DEV)
    check(w, x, torch.zeros(B, C, device=DEV), None, "log", tied, dy, None)
    doc = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    doc[:, T // 3:], doc[:, T // 3 + 5:T // 3 + 9] = 1, -1
    check(w, x, None, doc, "log", tied, dy, torch.zeros(B, C, device=DEV))
