"""64-bit reference of the MXFP4 layer with the bound of an evaluation that keeps sums, expert outputs and the combine
in fp32, whatever the call's size: every element is held to its own magnitude, not to its neighbours'."""
import torch

from mx_ref import U, _matmul, mx_values, scale_byte


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
        # |silu'| < 1.1; the exponential's argument g log2(e) is rounded, then three operations
        dh = (1.1 * dg) * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + h.abs() * (g.abs() + 8) * U
        hq, dq = mx_values(h, "mxfp6"), torch.zeros_like(h)
        top, dtop = (v.reshape(len(t), -1, 32).amax(-1, keepdim=True) for v in (h.abs(), dh))
        for s in (scale_byte((top - dtop).clamp_min(0), "mxfp6"), scale_byte(top + dtop, "mxfp6")):
            for v in (h - dh, h + dh):   # the codes that a value within its error of a border may take
                dq = torch.maximum(dq, (mx_values(v, "mxfp6", s) - hq).abs())
        o, do = _matmul(w2[e], hq, dq)
        a = tw[t, k].unsqueeze(1)
        y.index_add_(0, t, a * o)
        bound.index_add_(0, t, a.abs() * (do + (o.abs() + do) * (ids.shape[1] + 2) * U))
    fi = torch.finfo(dtype)
    return y, bound + (y.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
