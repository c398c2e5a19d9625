"""The expert layer with microscaled 4-bit weights and the router in front of it.

Three kinds of case, each the work that serving a mixture-of-experts model puts on one call:

* "router": scores of T tokens over E experts -> the K picks of every token and their weights (softmax or sigmoid
  scores, a selection bias, expert groups, renormalised and scaled weights);
* "quantize": rows of 16- or 32-bit values -> blocks of 32 that share a power-of-two scale (MXFP4: E2M1 elements,
  MXFP6: E2M3), and back to the values they stand for;
* "layer": y[t] = sum_k w[t,k] * W2[e] (silu(W1[e] x) * (W3[e] x)) with MXFP4 weights; x and the intermediate are
  quantized to MXFP6.  With "scores" the call starts from the router's logits.

Sizes are those of the repository's configurations (H=2048 I=768 E=128 top-8; H=2048 I=512 top-10) and generic ones.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MANTISSA = {"mxfp4": 1, "mxfp6": 3}


def _router(name, T, E, K, score="sigmoid", bias=True, groups=1, top_groups=1, group_top=2, renorm=True, scale=1.0,
            dtype="fp32"):
    c = {"op": "router", "tokens": T, "E": E, "top_k": K, "score": score, "bias": bias, "groups": groups,
         "top_groups": top_groups, "group_top": group_top, "renorm": renorm, "scale": scale, "dtype": dtype}
    return {"name": name, **c} if name else c


def _quantize(name, rows, cols, fmt, dtype="bf16"):
    c = {"op": "quantize", "rows": rows, "cols": cols, "format": fmt, "dtype": dtype}
    return {"name": name, **c} if name else c


def _layer(name, T, E, H, I, K, act="bf16", routing="uniform", call="op"):
    """routing: "uniform", or "skewed" (expert popularity as rank^-1.2); call: "op", or "scores" (from logits)."""
    c = {"op": "layer", "tokens": T, "E": E, "H": H, "I": I, "top_k": K, "dtype": act, "routing": routing, "call": call}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's next token: grouped sigmoid router of a large expert pool
        _router("router_1", 1, 256, 8, groups=8, top_groups=4, scale=2.5),
        # a running batch of a small pool, softmax scores, weights as they are
        _router("router_37_softmax", 37, 60, 6, score="softmax", bias=False, renorm=False, dtype="bf16"),
        # prompts of a whole batch
        _router("router_16384", 16384, 256, 8, groups=8, top_groups=4, scale=2.5, dtype="bf16"),
        # the hidden states of a few running sequences
        _quantize("quantize_act_5", 5, 2048, "mxfp6"),
        # the hidden states of a prefill chunk
        _quantize("quantize_act_8191", 8191, 2048, "mxfp6", dtype="fp16"),
        # a checkpoint's gate and up weights of 64 experts on their way into a handle
        _quantize("quantize_weights", 64 * 1536, 2048, "mxfp4"),
        # one user's next token
        _layer("layer_decode_1", 1, 128, 2048, 768, 8),
        # a small batch of users, from the router's logits
        _layer("layer_decode_8_scores", 8, 128, 2048, 768, 8, call="scores"),
        # some dozens of running sequences, top-10 of narrow experts
        _layer("layer_batch_45", 45, 128, 2048, 512, 10),
        # a short prompt whose tokens crowd on some experts
        _layer("layer_prompt_333_skewed", 333, 128, 2048, 768, 8, act="fp16", routing="skewed"),
        # a full prefill chunk
        _layer("layer_prefill_4096", 4096, 128, 2048, 768, 8),
        # the same of fewer, wider experts, an intermediate size that is no multiple of 128
        _layer("layer_prefill_wide", 5000, 64, 4096, 1440, 6),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["router", "quantize", "layer", "layer"])
    if op == "router":
        groups = rng.choice([1, 1, 4, 8])
        E = groups * log_int(max(2, 16 // groups), 512 // groups)
        top = rng.randint(1, groups)
        K = rng.randint(1, min(16, top * (E // groups)))
        return _router(None, log_int(1, 16384), E, K, score=rng.choice(["sigmoid", "softmax"]),
                       bias=rng.random() < 0.6, groups=groups, top_groups=top, group_top=rng.randint(1, 2),
                       renorm=rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 2.5, 16.0]),
                       dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "quantize":
        rows = log_int(1, 64 * 1536)
        return _quantize(None, rows, 32 * log_int(1, min(256, 2 * 1536 * 2048 // rows)), rng.choice(["mxfp4", "mxfp6"]),
                         dtype=rng.choice(["bf16", "fp16", "fp32"]))
    E = log_int(8, 256)
    H, I, K = 64 * log_int(8, 64), 32 * log_int(8, 64), rng.randint(1, min(E // 2, 10))
    while E * H * I > 128 * 2048 * 768:
        E, H, I = max(8, E * 3 // 4), max(512, H * 7 // 8 // 64 * 64), max(256, I * 7 // 8 // 32 * 32)
    K = min(K, E // 2)
    T = log_int(1, 4096)
    while T * K * H * I > 4096 * 8 * 2048 * 768:
        T = max(1, T // 2 - rng.randint(0, 1))
    call = rng.choice(["op", "op", "scores"])
    return _layer(None, T, E, H, I, K, act=rng.choice(["bf16", "bf16", "fp16"]), call=call,
                  routing="uniform" if call == "scores" else rng.choice(["uniform", "skewed"]))


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 17 + what)


def _scores_inputs(c, seed):
    """Router logits of some spread over the experts, and a bias as balancing leaves it."""
    g = _gen(seed, 0)
    logits = torch.randn(c["tokens"], c["E"], generator=g, device="cuda") * 1.5
    bias = torch.randn(c["E"], generator=g, device="cuda") * 0.05
    return logits, bias


def _inputs(c, seed):
    """What the call is given, in its types: the same for the plain form, the kernels and the 64-bit results."""
    if c["op"] == "router":
        logits, bias = _scores_inputs(c, seed)
        return {"logits": logits.to(DTYPE[c["dtype"]]), "bias": bias if c["bias"] else None}
    if c["op"] == "quantize":
        g = _gen(seed, 1)
        x = torch.randn(c["rows"], c["cols"], generator=g, device="cuda")
        if c["format"] == "mxfp6":   # hidden states: channels of unequal size
            x *= torch.exp(0.7 * torch.randn(c["cols"], generator=g, device="cuda"))
        else:
            x *= 0.02
        return {"x": x.to(DTYPE[c["dtype"]])}
    T, E, H, I, K = (c[k] for k in ("tokens", "E", "H", "I", "top_k"))
    g = _gen(seed, 2)
    x = torch.randn(T, H, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(H, generator=g, device="cuda"))
    d = {"x": x.to(DTYPE[c["dtype"]])}
    logits, bias = _scores_inputs(c, seed)
    if c["call"] == "scores":
        d["logits"], d["bias"] = logits, bias
    else:
        if c["routing"] == "skewed":   # rank^-1.2 popularity, K different experts a token (Gumbel top-k)
            rank = torch.randperm(E, generator=g, device="cuda") + 1
            u = torch.rand(T, E, generator=g, device="cuda").clamp_min(1e-20)
            logits = -1.2 * torch.log(rank.float()) - torch.log(-torch.log(u))
        val, ids = torch.topk(logits, K, dim=-1)
        d["ids"], d["w"] = ids.to(torch.int32), torch.softmax(val, dim=-1)
    for name, N, C in (("w13", 2 * I, H), ("w2", H, I)):
        codes, scales = [], []
        step = max(1, (1 << 26) // (N * C))   # experts at a time
        for e in range(0, E, step):
            a, b = _mxfp4_codes(torch.randn(min(step, E - e), N, C, generator=g, device="cuda") * 0.02)
            codes.append(a)
            scales.append(b)
        d[name], d[name + "_s"] = torch.cat(codes), torch.cat(scales)
    return d


def _mxfp4_codes(w):
    """[..., C] -> E2M1 codes [..., C/2] (element 2i in the low half of byte i) and E8M0 scales [..., C/32]."""
    b = w.reshape(*w.shape[:-1], -1, 32)
    e = _shared_exponent(b.abs().amax(-1), 1)
    v = torch.ldexp(b, -e.unsqueeze(-1))
    m = _round_element(v.abs(), 1)
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m * 0.5 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(*w.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def prepare(case, seed):
    c = case
    s = {"case": c, **_inputs(c, seed)}
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe-ascend-opt_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import nanovllm_moe
        nanovllm_moe.load()
        if c["op"] == "layer":   # the handle holds the weights from here on, as in a serving program
            h = torch.classes.nanovllm.MoEInfer(c["E"], c["H"], c["I"], 3)
            h.store_mxfp4_repack(s.pop("w13"), s.pop("w13_s"), s.pop("w2"), s.pop("w2_s"))
            s["handle"] = h
    return s


# ---------------------------------------------------------------------------------------------- plain form

def _shared_exponent(amax, mantissa):
    """The exponent of amax rounded to the element's mantissa bits, less the elements' largest exponent, 2."""
    m, e = torch.frexp(amax)   # amax = m 2^e, m in [0.5, 1)
    up = m >= 1 - 2.0 ** -(mantissa + 2)   # rounds to 1, the next power of two
    return torch.where(amax > 0, (e - 1 + up.to(e.dtype) - 2).clamp_min(-121), -121)


def _round_element(a, mantissa):
    """a >= 0 in units of the block's scale -> the nearest element value, ties to the even mantissa."""
    step = torch.where(a < 2, 1.0, torch.where(a < 4, 2.0, 4.0)) * 2.0 ** -mantissa
    return torch.round(a / step) * step


def _mx_values(x, fmt):
    b = x.reshape(*x.shape[:-1], -1, 32)
    e = _shared_exponent(b.abs().amax(-1, keepdim=True), MANTISSA[fmt])
    v = torch.ldexp(b, -e)
    return torch.ldexp(torch.copysign(_round_element(v.abs(), MANTISSA[fmt]), v), e).reshape(x.shape)


def _picks(logits, bias, c):
    """ids and weights; in 64 bits, since two scores may lie nearer to each other than 32 bits tell."""
    T, E, G, K = c["tokens"], c["E"], c["groups"], c["top_k"]
    v = logits.double()
    if c["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-v))
    else:
        p = torch.exp(v - v.amax(-1, keepdim=True))
        s = p / p.sum(-1, keepdim=True)
    choice = s if bias is None else s + bias.double()
    if c["top_groups"] < G:
        grouped = choice.reshape(T, G, E // G)
        rank = torch.sort(grouped, dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
        keep = torch.zeros(T, G, dtype=torch.bool, device=v.device)
        keep.scatter_(1, order[:, :c["top_groups"]], True)
        choice = torch.where(keep.unsqueeze(-1), grouped, -math.inf).reshape(T, E)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :K]
    w = torch.gather(s, 1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.to(torch.int32), (w * c["scale"]).float()


def _weights(codes, scales):
    """MXFP4 codes and scales -> values, 32 bits."""
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([half, -half])
    i = torch.arange(256, device=codes.device)
    pairs = torch.stack([table[i & 15], table[i >> 4]], -1)   # byte -> its two elements
    v = pairs[codes.int()].reshape(*scales.shape, 32)
    return (v * torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127).unsqueeze(-1)).reshape(
        *codes.shape[:-1], -1)


def _mlp(x, w13, w2):
    """x [B,M,H], w13 [B,2I,H], w2 [B,H,I] -> [B,M,H]."""
    g, u = torch.bmm(x, w13.transpose(1, 2)).chunk(2, dim=-1)
    h = _mx_values(g / (1 + torch.exp(-g)) * u, "mxfp6")
    return torch.bmm(h, w2.transpose(1, 2))


def _experts(s, ids, w):
    c = s["case"]
    T, E, H, K = c["tokens"], c["E"], c["H"], c["top_k"]
    x = _mx_values(s["x"].float(), "mxfp6")
    flat = ids.reshape(-1).long()
    if T * K <= 64:   # few pairs: each with its own expert's weights
        pairs = x.repeat_interleave(K, 0).unsqueeze(1)
        out = _mlp(pairs, _weights(s["w13"][flat], s["w13_s"][flat]), _weights(s["w2"][flat], s["w2_s"][flat]))
        out = out.reshape(T, K, H)
    else:             # every expert with the rows that are routed to it, padded to the longest
        order = torch.argsort(flat, stable=True)
        count = torch.bincount(flat, minlength=E)
        at = torch.arange(T * K, device=x.device) - (torch.cumsum(count, 0) - count)[flat[order]]
        rows = torch.zeros(E, int(count.max()), H, device=x.device)
        rows[flat[order], at] = x[order // K]
        res = _mlp(rows, _weights(s["w13"], s["w13_s"]), _weights(s["w2"], s["w2_s"]))
        out = torch.empty(T * K, H, device=x.device)
        out[order] = res[flat[order], at]
        out = out.reshape(T, K, H)
    return (out * w.unsqueeze(-1)).sum(1).to(s["x"].dtype)


LAYER_ROUTER = {"score": "sigmoid", "groups": 1, "top_groups": 1, "group_top": 2, "renorm": True, "scale": 1.0}


def run(state):
    s, c = state, state["case"]
    if own:
        ops = torch.ops.nanovllm
        if c["op"] == "router":
            return ops.moe_topk_scores(s["logits"], c["top_k"], s["bias"], c["score"], c["groups"], c["top_groups"],
                                       c["group_top"], c["renorm"], c["scale"])
        if c["op"] == "quantize":
            codes, scales = ops.mx_quantize(s["x"], c["format"])
            return ops.mx_dequantize(codes, scales, c["format"], s["x"].dtype)
        if c["call"] == "scores":
            return ops.moe_forward_scores(s["x"], s["logits"], c["top_k"], s["bias"], "sigmoid", 1, 1, 2, True, 1.0,
                                          s["handle"])
        return ops.moe_forward(s["x"], s["ids"], s["w"], s["handle"])
    if c["op"] == "router":
        return _picks(s["logits"], s["bias"], c)
    if c["op"] == "quantize":
        return _mx_values(s["x"].float(), c["format"]).to(s["x"].dtype)
    if c["call"] == "scores":
        return _experts(s, *_picks(s["logits"], s["bias"], {**c, **LAYER_ROUTER}))
    return _experts(s, s["ids"], s["w"])


def work(case):
    c = case
    if c["op"] == "router":   # about 60 operations a logit: an exponential in 64 bits, the bias, a place in the order
        T, E = c["tokens"], c["E"]
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": T * E * size + T * c["top_k"] * 8 + (4 * E if c["bias"] else 0), "flops": 60.0 * T * E}
    if c["op"] == "quantize":   # values in, codes and scales out and in again, values out
        n = c["rows"] * c["cols"]
        held = n * (4 + 2 * (c["format"] == "mxfp6")) / 8 + n / 32
        return {"bytes": n * (8 if c["dtype"] == "fp32" else 4) + 2 * held, "flops": 6.0 * n}
    T, K, E, H, I = (c[k] for k in ("tokens", "top_k", "E", "H", "I"))
    used = E * (1.0 - (1.0 - K / E) ** T)   # experts that some token is routed to
    if c["routing"] == "skewed":   # a random order has the same sum over experts
        p = [r ** -1.2 for r in range(1, E + 1)]
        used = sum(1.0 - (1.0 - min(1.0, K * v / sum(p))) ** T for v in p)
    route = 4 * T * E + 4 * E if c["call"] == "scores" else 8 * T * K
    return {"bytes": used * 3 * H * I * 17 / 32 + 4 * T * H + route, "flops": 6.0 * T * K * H * I}


# ---------------------------------------------------------------------------------------------- 64 bits

def _grid(fmt):
    """The element values of a format that are not negative, ascending: (1 + m/2^M) 2^(e-1), and m/2^M for e = 0."""
    M = MANTISSA[fmt]
    small = [m / 2 ** M for m in range(2 ** M)]
    return small + [(1 + v) * 2 ** (e - 1) for e in (1, 2, 3) for v in small]


def _exact_mx(x, fmt):
    x = x.double().reshape(-1, 32)
    top = x.abs().max(dim=1, keepdim=True).values
    grid = torch.tensor(_grid(fmt), dtype=torch.float64, device=x.device)
    limit = (grid[-1] + 2 ** (2 - MANTISSA[fmt]) / 2).item()   # what rounds to more than the largest element
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** -140)))
    # log2 may be one off at powers of two
    e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double() - 2
    e = (e + (top >= limit * torch.exp2(e))).clamp_min(-121)
    a = (x / torch.exp2(e)).abs()
    hi = torch.searchsorted(grid, a).clamp_(1, len(grid) - 1)
    lo = hi - 1
    below, above = a - grid[lo], grid[hi] - a
    pick = torch.where(below < above, lo, torch.where(above < below, hi, lo + lo % 2))   # a tie: the even code
    return torch.sign(x) * grid[pick] * torch.exp2(e)


def _exact_dequant(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).long()
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double())) * (1 - 2 * (c >> 3).double())
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


def _exact_picks(logits, bias, c):
    v = logits.double()
    s = torch.sigmoid(v) if c["score"] == "sigmoid" else torch.softmax(v, dim=-1)
    choice = s.clone() if bias is None else s + bias.double()
    T, E, G = c["tokens"], c["E"], c["groups"]
    best = torch.topk(choice.view(T, G, E // G), min(c["group_top"], E // G), dim=-1).values.sum(-1)
    other, this = best.unsqueeze(1), best.unsqueeze(2)
    # [this, other]: a tie goes to the lower index
    first = torch.ones(G, G, dtype=torch.bool, device=v.device).tril(-1)
    ahead = ((other > this) | ((other == this) & first)).sum(-1)   # groups that come before each
    closed = (ahead >= c["top_groups"]).repeat_interleave(E // G, dim=1)
    choice[closed] = -math.inf
    ids = torch.argsort(-choice, dim=-1, stable=True)[:, :c["top_k"]]
    w = s.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.to(torch.int32), w * c["scale"]


def exact(case, seed):
    c = case
    d = _inputs(c, seed)
    if c["op"] == "router":
        return _exact_picks(d["logits"], d["bias"], c)
    if c["op"] == "quantize":
        rows = d["x"].reshape(c["rows"], c["cols"])
        step = max(1, (1 << 25) // c["cols"])
        return torch.cat([_exact_mx(rows[r:r + step], c["format"]).reshape(-1, c["cols"])
                          for r in range(0, c["rows"], step)])
    if c["call"] == "scores":
        ids, w = _exact_picks(d["logits"], d["bias"], {**c, **LAYER_ROUTER})
    else:
        ids, w = d["ids"], d["w"].double()
    x = _exact_mx(d["x"], "mxfp6").reshape(c["tokens"], c["H"])
    y = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        t, k = torch.nonzero(ids == e, as_tuple=True)
        gu = x[t] @ _exact_dequant(d["w13"][e], d["w13_s"][e]).t()
        g, u = gu[:, :c["I"]], gu[:, c["I"]:]
        h = _exact_mx(torch.nn.functional.silu(g) * u, "mxfp6").reshape(len(t), c["I"])
        y.index_add_(0, t, (h @ _exact_dequant(d["w2"][e], d["w2_s"][e]).t()) * w[t, k].unsqueeze(1))
    return y
