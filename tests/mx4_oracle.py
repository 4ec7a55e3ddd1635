"""The 4-bit microscaled format in float64, from its definition, on whatever device its inputs are."""

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
U = 2.0 ** -24  # half a step of fp32, relative


def exponents(top):
    """The block exponent e of a block's largest size (e = floor(log2 top) - 2, at least -127)."""
    frac, exp = torch.frexp(top.double())  # top = frac 2^exp, frac in [0.5, 1)
    return torch.where(top > 0, (exp - 3).clamp(min=-127), torch.full_like(exp, -127))


def level_index(ratio):
    """Index of the nearest level to sizes `ratio` (halfway: the even index)."""
    idx = torch.zeros(ratio.shape, dtype=torch.int64, device=ratio.device)
    for n in range(7):
        middle = 0.5 * (LEVELS[n] + LEVELS[n + 1])
        idx += (ratio > middle) if n % 2 == 0 else (ratio >= middle)
    return idx


def pow2(e):
    """2^e in float64 for whole e in [-1022, 1023], from its bits: torch.pow on the GPU is off by a rounding for some."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantize(x):
    """(level indices with sign bit uint8 [..., K], scale bytes uint8 [..., K/32])."""
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    clean = torch.where(bad, torch.zeros_like(b), b)
    e = exponents(clean.abs().amax(-1, keepdim=True))
    idx = level_index(clean.abs() / pow2(e)) + 8 * torch.signbit(clean)
    idx = torch.where(bad, torch.zeros_like(idx), idx)
    s = torch.where(bad, torch.full_like(e, 255), e + 127)
    return idx.flatten(-2).to(torch.uint8), s.squeeze(-1).to(torch.uint8)


def pack(idx):
    return idx[..., 0::2] | (idx[..., 1::2] << 4)


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)


def values(idx, s):
    """float64 values of level indices [..., K] and scale bytes [..., K/32 or more]."""
    table = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=idx.device)
    K = idx.shape[-1]
    s = s[..., :K // 32].long()
    f = torch.where(s == 255, torch.full(s.shape, float("nan"), dtype=torch.float64, device=s.device), pow2(s - 127))
    return (table[idx.long()].unflatten(-1, (-1, 32)) * f.unsqueeze(-1)).flatten(-2)


def silu(g):
    return g * torch.special.expit(g)


def product(a, w, counts):
    """(C, bound of fp32 accumulation) of grouped rows a [M, K] and weights w [G, N, K], float64: K products, exact in
    fp32 (two 2-bit significands), added in any order by sums that round to within a step (2 u) each."""
    out, err, lo = [], [], 0
    for g, n in enumerate(counts):
        r = a[lo:lo + n]
        out.append(r @ w[g].t())
        err.append(2 * a.shape[1] * U * (r.abs() @ w[g].t().abs()))
        lo += n
    return torch.cat(out), torch.cat(err)


def swiglu(c, e):
    """(act, bound) from gate | up columns: silu's slope is below 1.1; the hardware exponential of g log2(e) is off by
    (|g| + 2) 2^-23 relative, reciprocal and products by 2^-23 more."""
    g, u = c.chunk(2, -1)
    eg, eu = e.chunk(2, -1)
    s = silu(g)
    es = 1.1 * eg + s.abs() * (g.abs() + 6) * 2 * U
    return s * u, es * (u.abs() + eu) + s.abs() * eu + 2 * U * (s * u).abs()


def requantize(v, e):
    """(values of v as 4-bit blocks, how far those of anything within e of v may be from them)."""
    b, eb = v.unflatten(-1, (-1, 32)), e.unflatten(-1, (-1, 32))

    def at(x, exp):
        table = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
        return torch.copysign(table[level_index(x.abs() / pow2(exp))], x) * pow2(exp)

    top = b.abs()
    mid = at(b, exponents(top.amax(-1, keepdim=True)))
    far = torch.zeros_like(mid)
    for t in ((top + eb), (top - eb).clamp(min=0)):
        exp = exponents(t.amax(-1, keepdim=True))
        for x in (b - eb, b + eb):
            far = torch.maximum(far, (at(x, exp) - mid).abs())
    return mid.flatten(-2), far.flatten(-2)
