"""CPU: the 64-bit gated delta rule against its recurrence in closed form and its gradients against differences."""
import pytest
import torch

from oracle import delta as O
from _mixers_util import doc_ids, randn


def some(B=2, T=7, H=4, Hk=2, N=8, seed=0):
    z = lambda i, *s: randn(*s, seed=seed + i).double()
    return [z(1, B, T, Hk, N), z(2, B, T, Hk, N) / 3, z(3, B, T, H, N), -z(4, B, T, H).exp(), torch.sigmoid(z(5, B, T, H)), z(6, B, H, N, N)]


def test_one_token_and_one_channel():
    q, k, v, g, beta, s0 = some(1, 1, 1, 1, 8)
    out = O.gated_delta(q, k, v, g, beta, s0, scale=1.0)
    s = s0[0, 0] * g[0, 0, 0].exp()
    s = s - beta[0, 0, 0] * torch.outer(k[0, 0, 0], s.T @ k[0, 0, 0]) + beta[0, 0, 0] * torch.outer(k[0, 0, 0], v[0, 0, 0])
    assert torch.allclose(out["sT"][0, 0], s, atol=1e-12) and torch.allclose(out["y"][0, 0, 0], s.T @ q[0, 0, 0], atol=1e-12)


@pytest.mark.parametrize("kind", [None, "two", "padded", "one"])
def test_gradients_against_differences(kind):
    args = some()
    B, T = args[0].shape[:2]
    doc = None if kind is None else doc_ids(B, T, kind, seed=1)
    dy, dsT = randn(*args[2].shape, seed=8).double(), randn(*args[5].shape, seed=9).double()
    out = O.gated_delta(*args, doc=doc, dy=dy, dsT=dsT)

    def loss(z):
        o = O.gated_delta(*z, doc=doc)
        return float((o["y"] * dy).sum() + (o["sT"] * dsT).sum())
    for i, n in enumerate(("dq", "dk", "dv", "dg", "dbeta", "ds0")):
        way = randn(*args[i].shape, seed=20 + i).double()
        h = 1e-6
        ends = [loss([z + s * h * way if j == i else z for j, z in enumerate(args)]) for s in (1, -1)]
        assert abs((ends[0] - ends[1]) / (2 * h) - float((out[n] * way).sum())) < 1e-7 * (1 + abs(ends[0])), n


def test_documents_are_calls_of_their_own_and_padding_is_nothing():
    q, k, v, g, beta, s0 = some(1, 12)
    doc = torch.tensor([[0, 0, 0, -1, -1, 4, 4, 4, 4, 2, 2, -1]], dtype=torch.int32)
    out = O.gated_delta(q, k, v, g, beta, s0, doc)
    for lo, hi, s in ((0, 3, s0), (5, 9, None), (9, 11, None)):
        part = O.gated_delta(*(z[:, lo:hi] for z in (q, k, v, g, beta)), s)
        assert torch.allclose(out["y"][:, lo:hi], part["y"], atol=1e-12)
    assert torch.allclose(out["sT"], part["sT"], atol=1e-12) and not out["y"][:, 3:5].any()
