"""Helpers for the tests of the gated delta rule."""
import torch

from oracle.mixers import LEAST, TINY, UNIT
from _gpu_util import DEV
from _mixers_util import randn

# How far a kernel may be off beside its one rounding at the end.  Operands of matrix products are kept as two numbers of 8 bits, off by 2^-18 of them at most, and the
# product of the two second numbers, at most 2^-18 of the product, is left out: 3 2^-18 at most for each product, and its root mean square a third of that.  Four products
# follow each other at most (the state's reading, the triangular system, the state's writing, the output's reading), in sums whose terms
# have errors of either sign: 4 2^-18 relative to the root mean square of a result.
PAIRS = 2.0 ** -16
# ... and for a single element up to 16 of these: it may be the sum of terms that are larger than itself, and the largest of some 10^6 errors is five of their root mean squares.
SINGLE = 16
# Decays below fp32's least normal number, 2^-126, are 0 to the hardware's exponential, so that 2^-126 of a state or gradient (here below 2^6 in magnitude), over up to 2^20 tokens, may be
# lost: LEAST = 2^-100, as for the gated recurrence.


def inputs(B, T, H, Hk, N, dt, seed=0, slow=3.0):
    """q and k of length 1, the keys of a head around one direction; time constants around e^slow; the gradients of y and sT."""
    z = lambda i, *s: randn(*s, seed=seed + i)
    unit = lambda x: x / x.square().sum(-1, keepdim=True).sqrt()
    q, k, v = unit(z(1, B, T, Hk, N)), unit(z(2, B, T, Hk, N) + 0.7 * z(3, 1, 1, Hk, N)), z(4, B, T, H, N)
    g, beta = -torch.exp(1.2 * z(5, B, T, H) - slow), torch.sigmoid(z(6, B, T, H))
    return [x.to(dt).to(DEV) for x in (q, k, v, g, beta)], (0.3 * z(7, B, H, N, N)).to(DEV), z(8, B, T, H, N).to(dt).to(DEV), (0.3 * z(9, B, H, N, N)).to(DEV)


def near(name, got, want, steps=1.0):
    """got against the 64-bit value, by root mean square over the whole and element by element; `steps` times PAIRS beside the rounding of the type."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.detach().double() - want).abs()
    rms = float(want.square().mean().sqrt())
    u, tiny = UNIT[got.dtype], TINY[got.dtype]
    rounding = float((want.to(got.dtype).double() - want).square().mean().sqrt())
    have, may = float(off.square().mean().sqrt()), rounding * 1.05 + steps * PAIRS * rms + tiny + LEAST
    single = (off / (u * want.abs() + tiny + SINGLE * steps * PAIRS * torch.maximum(want.abs(), torch.tensor(rms, device=want.device)) + LEAST)).max() if off.numel() else 0.0
    print(f"  {name}: error {have:.3e} of {may:.3e}, an element at most {float(single):.3f} of its bound", flush=True)
    assert have <= may and float(single) <= 1.0, name
