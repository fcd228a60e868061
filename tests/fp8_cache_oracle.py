"""Plain statements in 64 bits of the paged cache of 8 bits, the append with rotation and the decode attention over it, token by token."""
import math

import torch

MAX = 448.0


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """float64 numbers of at most 464 to the nearest number that e4m3 holds, ties to the even one; others to NaN."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.pow(2.0, e - 3)
    r = torch.round(y / step) * step                  # half to even
    return torch.where(y.isfinite() & (r.abs() <= MAX), r, float("nan"))


def rotated32(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, fused: bool) -> torch.Tensor:
    """Rotation of rows [T, heads, D] as the operators round it: float32 products and sums, ``fused``: the second product is not rounded by itself."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half].float(), x[..., half:].float(), cos[:, None], sin[:, None]
    if not fused:
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([(a.double() * c.double() - (b * s).double()).float(), (b.double() * c.double() + (a * s).double()).float()], -1)


def scale_for(most: float) -> float:
    return 0.0 if most == 0 else max(2.0 ** -126, 2.0 ** math.ceil(math.log2(most / MAX)))


def append(x, codes, scale, slots):
    """x: float32 [T, kv_heads, D]; codes (float64 values), scale (float64): new ones."""
    codes, scale = codes.clone(), scale.clone()
    blocks, heads, size, _ = codes.shape
    rows = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * size:
            rows.setdefault(s // size, {})[s % size] = t
    for block, written in rows.items():
        for h in range(heads):
            new = {r: x[t, h].double() for r, t in written.items()}
            most = max(float(v[v.isfinite()].abs().max()) if v.isfinite().any() else 0.0 for v in new.values())
            old = 0.0 if 0 in written else float(scale[block, h])
            to = max(scale_for(most), old)
            if 0 not in written and to > old:
                for r in range(size):
                    if r not in written:
                        codes[block, h, r] = round_e4m3(codes[block, h, r] * (old / to))
            for r, v in new.items():
                codes[block, h, r] = round_e4m3(v / to) if to else torch.where(v.isfinite(), 0.0, float("nan")).double()
            scale[block, h] = to
    return codes, scale


def attend(q, k, ks, v, vs, tables, lens, scale, most=None):
    """float64 [B, H, D] and, for each (b, h), what bounds the error of 32-bit arithmetic: (largest sum of |q k| * scale, largest |v|)."""
    B, H, D = q.shape
    heads, size = k.shape[1], k.shape[2]
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, 2, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b]) if most is None else min(int(lens[b]), most)
        n = min(n, tables.shape[1] * size)
        if n <= 0:
            continue
        at = torch.arange(n)
        page, row = tables[b].long()[at // size], at % size
        for h in range(H):
            g = h // (H // heads)
            kk, vv = k[page, g, row].double() * ks[page, g].double()[:, None], v[page, g, row].double() * vs[page, g].double()[:, None]
            s = (kk @ q[b, h].double()) * scale
            out[b, h] = torch.softmax(s, 0) @ vv
            bound[b, h, 0] = (kk.abs() @ q[b, h].double().abs()).max() * scale
            bound[b, h, 1] = vv.abs().max()
    return out, bound


def tolerance(out, bound, D):
    """Half a step of bf16 of the result; a score is a sum of D exact products in 32 bits (each addition off by at most 2^-23 of the sum of magnitudes, chopped
    or rounded) times two factors; weights are then off by twice that and by 2^-14 for their exponential and their rounding to 16 bits or more."""
    score = (D + 16) * 2.0 ** -23 * bound[..., 0]
    return 2.0 ** -8 * out.abs() + ((2 * score + 2.0 ** -14) * bound[..., 1])[..., None]
