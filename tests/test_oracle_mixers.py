"""CPU: the 64-bit formulas of the gated recurrence and of attention, against differences, autograd and special cases."""
import math

import pytest
import torch

from oracle import mixers as O


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def _value(f, up):
    return sum(float((f[n][0] * g).sum()) for n, g in up.items())


def _differences(f, leaf, step=1e-5):
    g = torch.zeros_like(leaf)
    for i in range(leaf.numel()):
        flat = leaf.view(-1)
        keep = float(flat[i])
        flat[i] = keep + step
        hi = f()
        flat[i] = keep - step
        lo = f()
        flat[i] = keep
        g.view(-1)[i] = (hi - lo) / (2 * step)
    return g


@pytest.fixture(autouse=True)
def _fp64(monkeypatch):
    monkeypatch.setitem(O.UNIT, torch.float64, 2.0 ** -53)
    monkeypatch.setitem(O.TINY, torch.float64, 0.0)


@pytest.mark.parametrize("gate", ["sigmoid", "log"])
@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("packed", [False, True])
def test_recurrence_gradients_against_differences(gate, tied, packed):
    B, T, C = 2, 9, 3
    w, x, h0 = _rand(B, T, C, seed=1), _rand(B, T, C, seed=2), _rand(B, C, seed=3)
    if gate == "log":
        w = -w.abs()
    doc = torch.tensor([[0, 0, 1, 1, -1, 1, 2, -1, -1], [-1, 4, 4, 4, 3, 4, -1, -1, 4]], dtype=torch.int32) if packed else None
    dy, dhT = _rand(B, T, C, seed=4), _rand(B, C, seed=5)
    got = O.gated_recurrence(w, x, h0, doc, gate, tied, dy, dhT)
    f = lambda: _value(O.gated_recurrence(w, x, h0, doc, gate, tied), {"y": dy, "hT": dhT})
    for n, leaf in (("dw", w), ("dx", x), ("dh0", h0)):
        assert torch.allclose(got[n][0], _differences(f, leaf), rtol=1e-6, atol=1e-7), n


def test_recurrence_documents_are_separate_calls():
    T, C = 12, 4
    w, x = _rand(1, T, C, seed=6), _rand(1, T, C, seed=7)
    doc = torch.tensor([[3] * 5 + [-1] * 2 + [1] * 5], dtype=torch.int32)
    y = O.gated_recurrence(w, x, None, doc)["y"][0]
    for lo, hi in ((0, 5), (7, 12)):
        assert torch.equal(y[:, lo:hi], O.gated_recurrence(w[:, lo:hi], x[:, lo:hi])["y"][0])
    assert not y[:, 5:7].any()
    constant = O.gated_recurrence(torch.zeros(1, T, C, dtype=torch.float64), torch.ones(1, T, C, dtype=torch.float64))["y"][0]
    assert torch.allclose(constant[0, :, 0], 1 - 0.5 ** torch.arange(1, T + 1, dtype=torch.float64))


@pytest.mark.parametrize("how", ["plain", "cap", "slopes", "doc", "prefix", "all", "wide"])
def test_attention_gradients_against_differences(how):
    B, Tq, Tk, H, Hk, N = 2, 5, 7, 2, 1, 3
    q, k, v = _rand(B, Tq, H, N, seed=1), _rand(B, Tk, Hk, N, seed=2), _rand(B, Tk, Hk, N, seed=3)
    dy = _rand(B, Tq, H, N, seed=4)
    o = dict(doc=torch.tensor([[0, 0, 0, 0, 1, 1, -1], [2, 2, -1, 2, 2, 2, 0]], dtype=torch.int32) if how in ("doc", "all") else None,
             prefix=torch.tensor([3, 6], dtype=torch.int32) if how in ("prefix", "all") else None,
             slopes=torch.tensor([0.5, 0.1]) if how in ("slopes", "all") else None, cap=1.5 if how in ("cap", "all") else 0.0, scale=0.7, causal=how != "wide")
    got = O.attention(q, k, v, dy=dy, **o)
    f = lambda: _value(O.attention(q, k, v, **o), {"y": dy})
    for n, leaf in (("dq", q), ("dk", k), ("dv", v)):
        assert torch.allclose(got[n][0], _differences(f, leaf), rtol=1e-5, atol=1e-6), n
    if how in ("doc", "all"):
        assert not got["y"][0][0, -1].any() and not got["dq"][0][0, -1].any() and not got["dk"][0][0, -1].any()


def test_attention_with_one_key_and_with_equal_scores():
    v = _rand(1, 6, 1, 4, seed=1)
    z = torch.zeros(1, 6, 1, 4, dtype=torch.float64)
    y = O.attention(z, z, v)["y"][0]
    assert torch.allclose(y[0, :, 0], v[0, :, 0].cumsum(0) / torch.arange(1, 7, dtype=torch.float64)[:, None])
    assert torch.equal(O.attention(z[:, :1], z[:, :1], v[:, :1])["y"][0], v[:, :1])


def test_paged_attention_is_the_last_row_of_attention():
    B, T, H, Hk, N, page = 2, 11, 4, 2, 3, 4
    q, k, v = _rand(B, T, H, N, seed=1), _rand(B, T, Hk, N, seed=2), _rand(B, T, Hk, N, seed=3)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0])
    want = O.attention(q, k, v, slopes=slopes, cap=2.0)["y"][0][:, -1]
    table = torch.tensor([[5, 0, 3], [1, 2, 4]], dtype=torch.int32)
    kp, vp = (torch.full((6, page, Hk, N), math.nan, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        for t in range(T):
            kp[table[b, t // page], t % page], vp[table[b, t // page], t % page] = k[b, t], v[b, t]
    got = O.paged_attention(q[:, -1], kp, vp, table, torch.tensor([T, T]), slopes=slopes, cap=2.0)["y"][0]
    assert torch.allclose(got, want)
