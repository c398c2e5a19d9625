"""Expert products on rows sorted by expert, and products in 8-bit integers.

Four kinds of case:

* "grouped": y[r] = W[e] x[r] for the rows r of every expert e (16-bit weights; ragged numbers of rows, some of them 0);
* "train": the same with its gradients, dx[r] = W[e]^T dy[r] and dW[e] = sum_r dy[r] x[r]^T;
* "quantize": rows of 16- or 32-bit values -> int8 codes and a scale for each row, and back to the values they stand for;
* "int8": y[m,n] = xs[m] ws[n] sum_k x[m,k] w[n,k] (+ bias[n]) of int8 codes, one weight ("experts" 0: a plain linear
  layer) or one for each expert with ragged rows.

Rows behind the last expert's ("tail": pairs dropped by the router, or padding) give zeros.  Sizes are those of the
repository's configurations (H=2048 I=768 E=128 top-8; H=2048 I=512 top-10) and generic ones.
"""
from __future__ import annotations

import os
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _grouped(name, op, rows, E, N, K, dtype="bf16", top_k=8, routing="uniform", tail=0):
    """routing: "uniform", or "skewed" (expert popularity as rank^-1.2); rows: routed pairs, tail: rows behind them."""
    c = {"op": op, "rows": rows, "E": E, "N": N, "K": K, "dtype": dtype, "top_k": top_k, "routing": routing, "tail": tail}
    return {"name": name, **c} if name else c


def _quantize(name, rows, cols, dtype="bf16"):
    c = {"op": "quantize", "rows": rows, "cols": cols, "dtype": dtype}
    return {"name": name, **c} if name else c


def _int8(name, rows, N, K, E=0, dtype="bf16", bias=False, top_k=8, routing="uniform", tail=0):
    c = {"op": "int8", "rows": rows, "E": E, "N": N, "K": K, "dtype": dtype, "bias": bias, "top_k": top_k,
         "routing": routing, "tail": tail}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's next token through the gate and up weights of its 8 experts
        _grouped("grouped_decode_8", "grouped", 8, 128, 1536, 2048),
        # the down product of a prompt of 5000 tokens, wide experts, an inner size that is no multiple of 64 elements,
        # some experts crowded
        _grouped("grouped_prefill_wide", "grouped", 30000, 64, 4096, 1440, dtype="fp16", top_k=6, routing="skewed"),
        # fine-tuning a small layer: odd sizes, pairs beyond the experts' capacity dropped
        _grouped("train_small", "train", 333, 16, 520, 776, dtype="fp16", top_k=4, tail=27),
        # a training step of 4096 tokens, gate and up weights of 128 experts
        _grouped("train_4096", "train", 32768, 128, 1536, 2048),
        # a training step of few wide experts
        _grouped("train_few_wide", "train", 16384, 8, 4096, 4096, top_k=2, routing="skewed"),
        # the hidden states of a few running sequences
        _quantize("quantize_5", 5, 2048),
        # the hidden states of a prefill chunk
        _quantize("quantize_8191", 8191, 4096, dtype="fp16"),
        # one user's next token through a projection with a bias
        _int8("int8_linear_1", 1, 4096, 2048, bias=True),
        # some hundred running sequences, the vocabulary part of one card, logits in 32 bits
        _int8("int8_linear_200", 200, 19001, 2048, dtype="fp32"),
        # a prefill chunk through a wide projection
        _int8("int8_linear_8192", 8192, 8192, 4096),
        # some dozens of running sequences, top-10 of narrow experts
        _int8("int8_grouped_450", 450, 1024, 2048, E=128, top_k=10, dtype="fp16"),
        # a prefill chunk, gate and up weights of 128 experts
        _int8("int8_grouped_32768", 32768, 1536, 2048, E=128, tail=111),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    def size(lo, hi, step):
        n = log_int(lo, hi)
        return n if rng.random() < 0.15 else max(step, n // step * step)

    op = rng.choice(["grouped", "train", "quantize", "int8", "int8"])
    if op == "quantize":
        rows = log_int(1, 32768)
        return _quantize(None, rows, size(32, max(32, min(16384, 8191 * 4096 // rows)), 8),
                         dtype=rng.choice(["bf16", "fp16", "fp32"]))
    E = log_int(2, 256)
    N, K = size(64, 8192, 8), 16 * log_int(4, 512)
    while E * N * K > 128 * 1536 * 2048:
        E, N, K = max(2, E * 3 // 4), max(64, N * 7 // 8 // 8 * 8), max(64, K * 7 // 8 // 16 * 16)
    rows = log_int(1, 32768)
    while rows * N * K > 16384 * 4096 * 4096:
        rows = rows * 3 // 4
    top_k, routing = rng.randint(1, min(E, 10)), rng.choice(["uniform", "uniform", "skewed"])
    tail = rng.choice([0, 0, log_int(1, 300)])
    if op == "int8":
        E = rng.choice([0, E])
        return _int8(None, rows, N, K, E=E, dtype=rng.choice(["bf16", "fp16", "fp32"]), top_k=top_k, routing=routing,
                     bias=E == 0 and rng.random() < 0.5, tail=tail if E else 0)
    return _grouped(None, op, rows, E, N, K, dtype=rng.choice(["bf16", "bf16", "fp16"]), top_k=top_k, routing=routing,
                    tail=tail)


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 17 + what)


def _starts(c, g):
    """First row of every expert's rows, and the end of the last's: top_k different experts a token, all pairs sorted."""
    E, K = c["E"], min(c["top_k"], c["E"])
    u = torch.rand((c["rows"] + K - 1) // K, E, generator=g, device="cuda").clamp_min(1e-20)
    logits = -torch.log(-torch.log(u))
    if c["routing"] == "skewed":
        rank = torch.randperm(E, generator=g, device="cuda") + 1
        logits = logits - 1.2 * torch.log(rank.float())
    ids = torch.topk(logits, K, dim=-1).indices.reshape(-1)[:c["rows"]]
    counts = torch.bincount(ids, minlength=E)
    return torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)


def _codes(x):
    """[..., C] -> int8 codes and a scale for each row."""
    s = x.abs().amax(-1) / 127
    return torch.round(x / s.unsqueeze(-1)).to(torch.int8), s


def _hidden(rows, cols, g):
    """Hidden states: channels of unequal size."""
    return torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(
        0.7 * torch.randn(cols, generator=g, device="cuda"))


def _inputs(c, seed):
    """What the call is given, in its types: the same for the plain form, the kernels and the 64-bit results."""
    g = _gen(seed, 3)
    if c["op"] == "quantize":
        return {"x": _hidden(c["rows"], c["cols"], g).to(DTYPE[c["dtype"]])}
    N, K, M = c["N"], c["K"], c["rows"] + c["tail"]
    d = {"starts": _starts(c, g)} if c["E"] else {}
    if c["op"] == "int8":
        d["x"], d["xs"] = _codes(_hidden(M, K, g))
        shape = (c["E"], N, K) if c["E"] else (N, K)
        d["w"] = torch.empty(shape, dtype=torch.int8, device="cuda")
        d["ws"] = torch.empty(shape[:-1], device="cuda")
        for q, s in zip(d["w"], d["ws"]) if c["E"] else ((d["w"], d["ws"]),):
            v, t = _codes(torch.randn(N, K, generator=g, device="cuda") * 0.02)
            q.copy_(v)
            s.copy_(t)
        d["bias"] = torch.randn(N, generator=g, device="cuda") * 0.1 if c["bias"] else None
        return d
    dt = DTYPE[c["dtype"]]
    d["x"] = torch.randn(M, K, generator=g, device="cuda").to(dt)
    d["w"] = torch.empty(c["E"], N, K, dtype=dt, device="cuda")
    for w in d["w"]:
        w.copy_(torch.randn(N, K, generator=g, device="cuda") * 0.02)
    if c["op"] == "train":
        d["dy"] = (torch.randn(M, N, generator=g, device="cuda") * 0.01).to(dt)
    return d


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe-ascend-opt_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import nanovllm_moe
        nanovllm_moe.load()
        if case["op"] == "train":
            s["x"].requires_grad_()
            s["w"].requires_grad_()
    elif case["op"] != "quantize" and case["E"]:
        s["ends"] = s["starts"].tolist()   # a loop over experts needs the numbers of rows on the host
    return s


# ---------------------------------------------------------------------------------------------- plain form

def _spans(s):
    return [(e, a, b) for e, (a, b) in enumerate(zip(s["ends"][:-1], s["ends"][1:])) if b > a]


def _plain_grouped(s):
    x, w = s["x"], s["w"]
    y = torch.zeros(x.shape[0], w.shape[1], dtype=x.dtype, device=x.device)
    for e, a, b in _spans(s):
        y[a:b] = torch.mm(x[a:b].float(), w[e].float().t()).to(x.dtype)
    return y


def _plain_train(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for e, a, b in _spans(s):
        g = dy[a:b].float()
        dx[a:b] = torch.mm(g, w[e].float()).to(x.dtype)
        dw[e] = torch.mm(g.t(), x[a:b].float()).to(w.dtype)
    return _plain_grouped(s), dx, dw


def _plain_quantize(x):
    v = x.float()
    top = v.abs().amax(-1)
    s = (top.double() / 127).clamp_min(2.0 ** -126).float()
    q = torch.round(v.double() / s.double().unsqueeze(-1))   # 64 bits: a quotient next to a border between two codes
    return (q.float() * s.unsqueeze(-1)).to(x.dtype), s


def _plain_int8(x, xs, w, ws, bias, dtype):
    acc = torch.mm(x.double(), w.double().t())   # up to 2^31: more than 32-bit floats hold
    y = acc * xs.double().unsqueeze(1) * ws.double()
    return (y if bias is None else y + bias.double()).to(dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        ops = torch.ops.nanovllm
        if c["op"] == "grouped":
            return ops.moe_grouped_matmul(s["x"], s["w"], s["starts"])
        if c["op"] == "train":
            y = ops.moe_grouped_matmul(s["x"], s["w"], s["starts"])
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return y.detach(), dx, dw
        if c["op"] == "quantize":
            q, scales = ops.int8_quantize(s["x"])
            return ops.int8_dequantize(q, scales, s["x"].dtype), scales
        if c["E"]:
            return ops.moe_grouped_matmul_int8(s["x"], s["xs"], s["w"], s["ws"], s["starts"], DTYPE[c["dtype"]])
        return ops.int8_matmul(s["x"], s["xs"], s["w"], s["ws"], s["bias"], DTYPE[c["dtype"]])
    if c["op"] == "grouped":
        return _plain_grouped(s)
    if c["op"] == "train":
        return _plain_train(s)
    if c["op"] == "quantize":
        return _plain_quantize(s["x"])
    dt = DTYPE[c["dtype"]]
    if not c["E"]:
        return _plain_int8(s["x"], s["xs"], s["w"], s["ws"], s["bias"], dt)
    y = torch.zeros(s["x"].shape[0], c["N"], dtype=dt, device=s["x"].device)
    for e, a, b in _spans(s):
        y[a:b] = _plain_int8(s["x"][a:b], s["xs"][a:b], s["w"][e], s["ws"][e], None, dt)
    return y


def work(case):
    c = case
    if c["op"] == "quantize":   # values in, codes and scales out and in again, values out
        n = c["rows"] * c["cols"]
        return {"bytes": n * (8 if c["dtype"] == "fp32" else 4) + 2 * (n + 4 * c["rows"]), "flops": 4.0 * n}
    M, N, K, E = c["rows"], c["N"], c["K"], c["E"]
    used, top = 1, min(c["top_k"], E)
    if E:   # experts that some row is routed to
        p = [1.0] * E if c["routing"] == "uniform" else [r ** -1.2 for r in range(1, E + 1)]
        used = sum(1.0 - (1.0 - min(1.0, top * v / sum(p))) ** (M / top) for v in p)
    flops = 2.0 * M * N * K
    if c["op"] == "int8":
        out = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": used * N * (K + 4) + M * (K + 4) + (M + c["tail"]) * N * out + 4 * (E + N * c["bias"]),
                "flops": flops}
    rows = M + c["tail"]
    fwd = 2 * (used * N * K + M * K + rows * N) + 4 * E
    if c["op"] == "grouped":
        return {"bytes": fwd, "flops": flops}
    return {"bytes": fwd + 2 * (M * N + rows * K + E * N * K), "flops": 3 * flops}


# ---------------------------------------------------------------------------------------------- 64 bits

def _exact_codes(x):
    x = x.double()
    s = (x.abs().max(dim=-1, keepdim=True).values / 127).clamp(min=2.0 ** -126).float().double()
    below = torch.floor(x / s)
    rest = x - below * s - s / 2   # exact: what decides is its sign
    up = (rest > 0) | ((rest == 0) & (below.remainder(2) == 1))
    return (below + up.double()) * s, s.squeeze(-1)


def exact(case, seed):
    c = case
    d = _inputs(c, seed)
    if c["op"] == "quantize":
        return _exact_codes(d["x"])
    x, w = d["x"], d["w"]
    if not c["E"]:
        y = (x.double() * d["xs"].double()[:, None]) @ (w.double() * d["ws"].double()[:, None]).T
        return y if d["bias"] is None else y + d["bias"].double()
    row = torch.arange(x.shape[0], device=x.device)
    expert = torch.searchsorted(d["starts"].long(), row, right=True) - 1   # rows behind the last expert's: E
    y = torch.zeros(x.shape[0], c["N"], dtype=torch.float64, device=x.device)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros(w.shape if c["op"] == "train" else (0,), dtype=torch.float64, device=x.device)
    for e in range(c["E"]):
        r = torch.nonzero(expert == e).squeeze(1)
        v = x[r].double()
        if c["op"] == "int8":
            y[r] = (v * d["xs"][r].double()[:, None]) @ (w[e].double() * d["ws"][e].double()[:, None]).T
            continue
        y[r] = v @ w[e].double().T
        if c["op"] == "train":
            g = d["dy"][r].double()
            dx[r] = g @ w[e].double()
            dw[e] = g.T @ v
    return (y, dx, dw) if c["op"] == "train" else y
