"""Products with weights of 4 bits in 64 bits, how far a kernel of 32-bit sums may be from them, and matrices to try them on."""
import torch

GROUP = 128


def matrix(rows, width, seed, device="cpu"):
    """Codes of all 16 values and scales of unlike size and sign, laid out as the quantiser lays them out."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (rows, width), generator=g, dtype=torch.uint8)
    scale = torch.randn(rows, width // GROUP, generator=g) * 0.01 * torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g).float())
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(device), scale.half().to(device)


def wide(w, scale):
    """The matrix in 64 bits."""
    codes = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.float64, device=w.device)
    codes[:, 0::2], codes[:, 1::2] = (w & 15).double(), (w >> 4).double()
    return (codes - 8) * scale.double().repeat_interleave(GROUP, 1)


def product(x, w, scale, gated=False, widened=False):
    """(value, bound on the error of a bf16 result).  A sum of n numbers in 32 bits is off by at most n 2^-23 of the sum of their sizes, a group's 128 and those
    between the groups; weights rounded to fp16 (``widened``) add 2^-12 of it, the result's own rounding 2^-8 of the value (half a step: eps / 2)."""
    full, x = wide(w, scale), x.double()
    y, size = x @ full.t(), x.abs() @ full.abs().t()
    off = size * ((GROUP + x.shape[-1] // GROUP) * 2.0 ** -23 + (2.0 ** -12 if widened else 0.0))
    if gated:
        (g, u), (eg, eu) = y.chunk(2, -1), off.chunk(2, -1)
        act = torch.nn.functional.silu(g)
        # silu's slope is at most 1.1; the exponential is off by 2 + 1.16 |g| steps of 2^-23, quotient and products by half a step each
        y, off = act * u, 1.1 * eg * u.abs() + (act.abs() + 1.1 * eg) * eu + (act * u).abs() * (5 + 1.2 * g.abs()) * 2.0 ** -23
    return y, off + (y.abs() + off) * 2.0 ** -8 + 1e-30


def check(got, want):
    y, bound = want
    assert got.shape == y.shape and torch.isfinite(got).all()
    over = (got.double() - y).abs() - bound
    assert over.max() <= 0, f"off by {over.max().item():.3g} more than the bound at {over.argmax().item()}"
