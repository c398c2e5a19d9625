"""64-bit references of the products on rows sorted by expert and of the int8 row quantizer, with bounds that count
every rounding of the kernels."""
import torch


def spans(starts, M):
    """[(expert, first row, end)]: starts read as its running maximum within [0, M]."""
    out, at = [], 0
    v = [min(max(int(s), 0), M) for s in starts]
    at = v[0]
    for e, s in enumerate(v[1:]):
        end = max(at, s)
        out.append((e, at, end))
        at = end
    return out


def round_bound(exact, slack, dtype):
    """Error of a value that is off by `slack` and then rounded to dtype: half a step of it (subnormal steps at least)."""
    f = torch.finfo(dtype)
    return slack + (exact.abs() + slack) * (f.eps / 2) + f.smallest_normal * f.eps / 2


def sum_slack(mag, n):
    """A sum of n products in fp32, in any order: each of its n additions is off by at most a step, 2^-23, of a partial
    sum that is no larger than mag, the sum of the products' magnitudes (which are exact in fp32)."""
    return mag * (n * 2.0 ** -23)


def grouped(x, w, starts, dtype):
    """y[r] = W[e] x[r] -> (exact, bound)."""
    M, N = x.shape[0], w.shape[1]
    y = torch.zeros(M, N, dtype=torch.float64, device=x.device)
    slack = torch.zeros_like(y)
    for e, a, b in spans(starts, M):
        y[a:b] = x[a:b].double() @ w[e].double().t()
        slack[a:b] = sum_slack(x[a:b].double().abs() @ w[e].double().abs().t(), x.shape[1])
    return y, round_bound(y, slack, dtype)


def grouped_dx(dy, w, starts, dtype):
    return grouped(dy, w.transpose(1, 2), starts, dtype)


def grouped_dw(dy, x, starts, E, dtype):
    dw = torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    slack = torch.zeros_like(dw)
    for e, a, b in spans(starts, x.shape[0]):
        g, v = dy[a:b].double(), x[a:b].double()
        dw[e] = g.t() @ v
        slack[e] = sum_slack(g.abs().t() @ v.abs(), b - a)
    return dw, round_bound(dw, slack, dtype)


def int8_rows(x, xs, w, ws, bias, dtype):
    """Exact integer sum, then four fp32 roundings (the sum, times ws, times xs, plus bias) of 2^-24 each, then dtype's."""
    p = (x.double() @ w.double().t()) * ws.double() * xs.double().unsqueeze(1)
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if bias is None else bias.double()
    slack = (p.abs() + b.abs()) * (4 * 2.0 ** -24 * (1 + 2.0 ** -20))
    return p + b, round_bound(p + b, slack, dtype)


def int8_grouped(x, xs, w, ws, starts, dtype):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e, a, b in spans(starts, x.shape[0]):
        y[a:b], bound[a:b] = int8_rows(x[a:b], xs[a:b], w[e], ws[e], None, dtype)
    return y, bound


def quantize(x):
    """Codes and scales of rows, by the definition."""
    v = x.double()
    bad = ~torch.isfinite(v).all(-1)
    s = (v.nan_to_num(0.0, 0.0, 0.0).abs().amax(-1) / 127).clamp_min(2.0 ** -126).float()
    q = torch.round(v / s.double().unsqueeze(-1))
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q).to(torch.int8)
    return q, torch.where(bad, torch.full_like(s, float("nan")), s)


def within(got, exact, bound):
    """Largest error in units of its bound."""
    assert got.shape == exact.shape
    if got.numel() == 0:
        return 0.0
    d = (got.to(exact.device).double() - exact).abs()
    assert bool(torch.isfinite(d).all())
    return float(torch.where(d == 0, d, d / bound).max())   # a bound of 0: exactly zero
