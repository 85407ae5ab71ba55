"""Helpers for the tests of the gated recurrence, attention and paged attention."""
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def randn(*shape, seed, dtype=torch.float32, scale=1.0, shift=0.0):
    """The same values on every device."""
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + shift).to(dtype)


def within(name, got, want):
    """Every element of `got` is as near the 64-bit value as the oracle's bound says."""
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.detach().double() - value).abs()
    worst = float((off / bound).max())
    print(f"  {name}: largest error {float(off.max()):.3e}, at most {worst:.3f} of its bound", flush=True)
    assert bool((off <= bound).all()), f"{name}: {worst:.3f} times the bound (NaN: {bool(torch.isnan(off).any())})"


def doc_ids(B, T, kind, seed=0):
    """Documents of a packed batch: "two" documents a row, "many" short ones, "padded" rows (padding behind, before and between; one row
    nothing but padding), "one" token documents, "back": an id that comes back behind another one."""
    g = torch.Generator().manual_seed(seed)
    doc = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        if kind == "two":
            doc[b, int(torch.randint(0, T + 1, (1,), generator=g)):] = 7
        elif kind == "many":
            for c in torch.randint(0, T, (max(1, T // 13),), generator=g).tolist():
                doc[b, c:] += 1
        elif kind == "padded":
            cut = sorted(torch.randint(0, T + 1, (4,), generator=g).tolist())
            doc[b, cut[2]:] = 5
            doc[b, cut[3]:] = -1
            doc[b, :cut[0]] = -3
            doc[b, cut[1]:cut[2]] = -1
            if b == B - 1 and B > 1:
                doc[b] = -1
        elif kind == "one":
            doc[b] = torch.arange(T, dtype=torch.int32)
        else:
            doc[b] = (torch.arange(T) // 5 % 2).to(torch.int32) + 3
    return doc


def graph_of(call, side=None):
    """Captures `call` on a stream of its own, after two runs there."""
    side = side or torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    return graph, out
