"""GPU: the gated recurrence, attention and paged attention as a hybrid model uses them: a layer of each on packed documents in training, and
the same two layers token by token in serving.  Every stage is held to the 64-bit definition at the inputs that it got."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from oracle import mixers as O
from rwkv_cuda_amd import attention as A, gated_recurrence as G, paged_attention as PA
from _gpu_util import DEV
from _mixers_util import DT, doc_ids, graph_of, randn, within

pytestmark = pytest.mark.gpu

H, HK, N = 6, 2, 64
C = (H + 2 * HK) * N


def qkv(z):
    """Queries, keys and values as views of the recurrence's output."""
    z = z.view(*z.shape[:-1], H + 2 * HK, N)
    return z[..., :H, :], z[..., H:H + HK, :], z[..., H + HK:, :]


def layers(w, x, doc, slopes):
    z, _ = G.RUN_CUDA(w, x, doc=doc)
    return z, A.RUN_CUDA(*qkv(z), doc=doc, slopes=slopes, cap=20.0)


def some(B, T, dt, seed):
    return [z.to(dt).to(DEV) for z in (randn(B, T, C, seed=seed, shift=1.0), randn(B, T, C, seed=seed + 1, scale=2.0))] + [torch.exp2(-torch.arange(1.0, H + 1)).to(DEV)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,T,kind", [(2, 333, "two"), (3, 200, "padded"), (1, 1, "two"), (2, 1100, "many")])
def test_training_on_packed_documents(lib, dtype, B, T, kind):
    w, x, slopes = some(B, T, DT[dtype], 1)
    doc = doc_ids(B, T, kind, seed=2).to(DEV)
    leaves = [z.requires_grad_(True) for z in (w, x)]
    z, y = layers(*leaves, doc, slopes)
    z.retain_grad()
    dy = randn(B, T, H, N, seed=5).to(DT[dtype]).to(DEV)
    y.backward(dy)
    want = O.attention(*qkv(z.detach()), doc=doc, slopes=slopes, cap=20.0, dy=dy)
    got = dict(zip(("dq", "dk", "dv"), qkv(z.grad)), y=y)
    for n in want:
        within(n, got[n], want[n])
    want = O.gated_recurrence(w, x, doc=doc, dy=z.grad)
    for n, g in (("y", z), ("dw", w.grad), ("dx", x.grad)):
        within(n, g, want[n])


def test_token_by_token_after_a_prompt(lib):
    """Prompts of several lengths, packed to one width by padding, then tokens one by one, the step captured once and replayed; some sequences
    begin with nothing.  The rows are those of the whole sequences."""
    B, page, M, prompt, new = 5, 16, 8, (40, 0, 17, 16, 33), 12
    dt, T = torch.bfloat16, max(prompt)
    w, x, slopes = some(B, T, dt, 11)
    wn, xn, _ = some(B, new, dt, 21)
    doc = torch.where(torch.arange(T) < torch.tensor(prompt)[:, None], 0, -1).to(torch.int32).to(DEV)
    table = torch.randperm(B * M, generator=torch.Generator().manual_seed(3)).view(B, M).to(torch.int32).to(DEV)
    kp, vp = (torch.full((B * M, page, HK, N), float("nan"), device=DEV, dtype=dt) for _ in range(2))
    with torch.no_grad():
        z, h = G.RUN_CUDA(w, x, doc=doc)
        _, k, v = qkv(z)
        for b, n in enumerate(prompt):                                # the prompt's keys and values go to their pages
            for t in range(n):
                kp[table[b, t // page], t % page], vp[table[b, t // page], t % page] = k[b, t], v[b, t]
        lens = torch.tensor(prompt, dtype=torch.int32, device=DEV)
        tw, tx = wn[:, 0].clone(), xn[:, 0].clone()

        def step():
            z = G.STEP(tw, tx, h)
            q, k, v = (t.contiguous() for t in qkv(z))
            lens.add_(1)
            return z, PA.RUN_CUDA(q, kp, vp, table, lens, k=k, v=v, slopes=slopes, cap=20.0)
        keep = [t.clone() for t in (h, lens)]
        graph, (zg, yg) = graph_of(step)
        torch.cuda.synchronize()
        h.copy_(keep[0]), lens.copy_(keep[1])                          # (the runs before the capture wrote where the first tokens go again)
        zs, ys = [], []
        for i in range(new):
            tw.copy_(wn[:, i]), tx.copy_(xn[:, i])
            graph.replay()
            torch.cuda.synchronize()
            zs.append(zg.clone()), ys.append(yg.clone())
    zs, ys = torch.stack(zs, 1), torch.stack(ys, 1)
    for b, n in enumerate(prompt):
        want = O.gated_recurrence(torch.cat([w[b:b + 1, :n], wn[b:b + 1]], 1), torch.cat([x[b:b + 1, :n], xn[b:b + 1]], 1))
        within(f"z of sequence {b}", zs[b:b + 1], tuple(t[:, n:] for t in want["y"]))
        within(f"state of sequence {b}", h[b:b + 1], want["hT"])
        whole = torch.cat([z[b:b + 1, :n], zs[b:b + 1]], 1)
        within(f"y of sequence {b}", ys[b:b + 1], tuple(t[:, n:] for t in O.attention(*qkv(whole), slopes=slopes, cap=20.0)["y"]))


def test_checkpoint_and_saved_tensor_hooks(lib):
    """The gradients under a checkpoint without re-entry are those without, and every saved tensor is unpacked once a backward."""
    w, x, slopes = some(2, 150, torch.bfloat16, 31)
    doc = doc_ids(2, 150, "two", seed=4).to(DEV)
    leaves = [z.requires_grad_(True) for z in (w, x)]
    run = lambda w, x: layers(w, x, doc, slopes)[1]
    grads = lambda y: torch.autograd.grad(y, leaves, torch.ones_like(y))
    want = grads(run(*leaves))
    assert all(torch.equal(a, b) for a, b in zip(want, grads(checkpoint(run, *leaves, use_reentrant=False))))
    count = {}

    def pack(z):
        count[len(count)] = 0
        return len(count) - 1, z

    def unpack(p):
        count[p[0]] += 1
        return p[1]
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = run(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, grads(y)))
    assert count and all(n == 1 for n in count.values()), count


def test_what_is_written_in_place_is_found_out_by_a_graph_that_saved_it(lib):
    w, x, _ = some(2, 3, torch.float32, 41)
    h = torch.ones(2, C, device=DEV)
    leaf = h.clone().requires_grad_(True)
    out = (leaf * h).sum()
    with torch.no_grad():
        G.STEP(w[:, 0], x[:, 0], h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()
    kp, vp = (torch.zeros(2, 16, HK, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    leaf = kp.clone().requires_grad_(True)
    out = (leaf * kp).sum()
    z = torch.zeros(2, HK, N, device=DEV, dtype=torch.bfloat16)
    table, lens = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    PA.RUN_CUDA(z, kp, vp, table, lens)                               # reads only
    out.backward(retain_graph=True)
    PA.RUN_CUDA(z, kp, vp, table, lens, k=z, v=z)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_in_inference_mode(lib):
    w, x, slopes = some(2, 20, torch.bfloat16, 51)
    with torch.no_grad():
        want = layers(w, x, None, slopes)
    with torch.inference_mode():
        got = layers(w, x, None, slopes)
        z, h = G.RUN_CUDA(w[:, :-1], x[:, :-1])
        kp, vp = (torch.zeros(4, 16, HK, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device=DEV)
        for t in range(20):
            last = G.STEP(w[:, -1], x[:, -1], h) if t == 19 else z[:, t]
            q, k, v = (u.contiguous() for u in qkv(last))
            y = PA.RUN_CUDA(q, kp, vp, table, torch.full((2,), t + 1, dtype=torch.int32, device=DEV), k=k, v=v, slopes=slopes, cap=20.0)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    within("y", y[:, None], tuple(t[:, -1:] for t in O.attention(*qkv(torch.cat([z, last[:, None]], 1)), slopes=slopes, cap=20.0)["y"]))


def test_document_ids_at_their_ends(lib):
    """The largest id, and one that follows it."""
    B, T = 2, 140
    w, x, slopes = some(B, T, torch.bfloat16, 61)
    doc = torch.full((B, T), 2 ** 31 - 1, dtype=torch.int32)
    doc[0, 30:90] = 0
    doc[1, 100:] = -2 ** 31
    doc = doc.to(DEV)
    with torch.no_grad():
        z, y = layers(w, x, doc, slopes)
    within("z", z, O.gated_recurrence(w, x, doc=doc)["y"])
    within("y", y, O.attention(*qkv(z), doc=doc, slopes=slopes, cap=20.0)["y"])


def test_inference_tensors_are_not_written_outside_of_inference_mode(lib):
    """torch refuses to write them there, and so do these; nothing has been written when they do."""
    with torch.inference_mode():
        h = torch.ones(2, C, device=DEV)
        kp, vp = (torch.zeros(2, 16, HK, N, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w, x, _ = some(2, 3, torch.float32, 71)
    z = torch.ones(2, HK, N, device=DEV, dtype=torch.bfloat16)
    table, lens = torch.tensor([[0], [1]], dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        for call in (lambda: G.STEP(w[:, 0], x[:, 0], h), lambda: G.STEP(w[:, 0], x[:, 0], torch.zeros(2, C, device=DEV), out=h),
                     lambda: PA.RUN_CUDA(z, kp, vp, table, lens, k=z, v=z), lambda: PA.RUN_CUDA(z, kp.clone(), vp, table, lens, k=z, v=z)):
            with pytest.raises(AssertionError, match="inference"):
                call()
        torch.cuda.synchronize()
        assert bool((h == 1).all()) and not kp.any() and not vp.any()
        PA.RUN_CUDA(z, kp, vp, table, lens)                          # reading is another matter
