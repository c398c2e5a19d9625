"""64-bit references of the MX formats and of the MXFP4 layer, with bounds.

The layer's reference returns, beside y, how far an fp32 evaluation may be
from it: every rounding counted, and for each intermediate value that lies
within its own error of a border between two MXFP6 codes, the step to the
other code."""
import torch

MANTISSA = {"mxfp4": 1, "mxfp6": 3}
BITS = {"mxfp4": 4, "mxfp6": 6}


def grid(fmt):
    """Element magnitudes in code order."""
    m = MANTISSA[fmt]
    low = [i / 2 ** m for i in range(2 ** m)]
    return torch.tensor(low + [(1 + v) * 2.0 ** e for e in (0, 1, 2) for v in low], dtype=torch.float64)


def scale_byte(amax, fmt):
    """The E8M0 byte for blocks of largest magnitude amax (finite, 64 bits)."""
    g = grid(fmt)
    limit = g[-1] + (g[-1] - g[-2]) / 2          # what rounds past the largest element
    s = torch.full_like(amax, 6, dtype=torch.float64)
    for b in range(7, 254):                      # the smallest scale that holds the block
        s = torch.where(amax >= limit * 2.0 ** (s - 127), torch.full_like(s, b), s)
    return s


def codes_of(x, s, fmt):
    """Magnitude codes of x (64 bits) under scale bytes s, by search of the nearest grid value, ties to the even code."""
    g = grid(fmt)
    a = (x / 2.0 ** (s - 127)).abs()
    hi = torch.searchsorted(g, a.contiguous()).clamp(1, len(g) - 1)
    lo = hi - 1
    d0, d1 = a - g[lo], g[hi] - a
    return torch.where(d0 < d1, lo, torch.where(d1 < d0, hi, torch.where(lo % 2 == 0, lo, hi)))


def mx_values(x, fmt, s=None):
    """x [..., C] (64 bits, finite) rounded to the format, with its scales or those given [..., C/32, 1]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    if s is None:
        s = scale_byte(b.abs().amax(-1, keepdim=True), fmt)
    return (torch.sign(b) * grid(fmt)[codes_of(b, s, fmt)] * 2.0 ** (s - 127)).reshape(x.shape)


def unpack(codes, fmt):
    """uint8 codes -> element codes, bit by bit."""
    bits = (codes.to(torch.int64).unsqueeze(-1) >> torch.arange(8)) & 1
    e = bits.reshape(*codes.shape[:-1], -1, BITS[fmt])
    return (e << torch.arange(BITS[fmt])).sum(-1)


def dequant(codes, scales, fmt):
    c = unpack(codes, fmt)
    top = 1 << (BITS[fmt] - 1)
    v = grid(fmt)[c & (top - 1)] * (1 - 2.0 * ((c & top) != 0))
    return v * 2.0 ** (scales.double() - 127).repeat_interleave(32, dim=-1)


U = 2.0 ** -23   # a sum's rounding, truncation allowed


def _matmul(w, x, dx=None):
    """x @ w.T and a bound of its fp32 error: a rounding for each group of 8 products and for each of the (at most
    8) parts of K that are added up, and what the inputs' error dx carries along."""
    mag = x.abs() @ w.abs().t()
    err = (x.shape[1] / 8 + x.shape[1] / 128 + 32) * U * mag
    if dx is not None:
        err = err + dx @ w.abs().t()
    return x @ w.t(), err


def layer(x, ids, tw, w13, w2, dtype):
    """y [T, H] and its bound, from x [T, H], ids, weights [T, K] and dequantized projections, all 64 bits."""
    T, H = x.shape
    E, I = w13.shape[0], w13.shape[1] // 2
    xq = mx_values(x, "mxfp6")
    y, bound = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if not len(t):
            continue
        gu, dgu = _matmul(w13[e], xq[t])
        g, u, dg, du = gu[:, :I], gu[:, I:], dgu[:, :I], dgu[:, I:]
        h = g * torch.sigmoid(g) * u
        s = (g * torch.sigmoid(g)).abs()
        # |silu'| < 1.1; the exponential's argument g log2(e) is rounded, then three operations
        dh = (1.1 * dg) * (u.abs() + du) + s * du + h.abs() * (g.abs() + 8) * U
        blocks = h.reshape(len(t), -1, 32)
        top, dtop = blocks.abs().amax(-1, keepdim=True), dh.reshape(len(t), -1, 32).amax(-1, keepdim=True)
        hq = mx_values(h, "mxfp6")
        dq = torch.zeros_like(h)
        for sb in (scale_byte((top - dtop).clamp_min(0), "mxfp6"), scale_byte(top + dtop, "mxfp6")):
            for v in (h - dh, h + dh):
                dq = torch.maximum(dq, (mx_values(v, "mxfp6", sb) - hq).abs())
        o, do = _matmul(w2[e], hq, dq)
        # expert outputs may be held in 16 bits relative to the largest of 64 columns
        top = (o.abs() + do).reshape(len(t), -1, 64).amax(-1, keepdim=True)
        do = do + (top * 2.0 ** -15).expand(-1, -1, 64).reshape(o.shape)
        a = tw[t, k].unsqueeze(1)
        y.index_add_(0, t, a * o)
        bound.index_add_(0, t, a.abs() * (do + (o.abs() + do) * (ids.shape[1] + 2) * U))
    fi = torch.finfo(dtype)
    return y, bound + (y.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2


def within(got, ref, bound):
    """The worst ratio of error to bound."""
    return float(((got.double() - ref).abs() / bound).max())
