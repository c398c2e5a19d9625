"""Plain 64-bit score router: one token and one expert at a time."""
import math


def route(logits, bias, K, sigmoid, n_group, topk_group, group_top, renorm, scale):
    """logits: a list of E numbers; bias: a list or None -> (ids, weights)."""
    E = len(logits)
    if sigmoid:
        s = [0.0 if l == -math.inf else 1.0 if l == math.inf else 1 / (1 + math.exp(-l)) if l > -700 else 0.0
             for l in logits]
        s = [math.nan if math.isnan(l) else v for l, v in zip(logits, s)]
    else:
        m = max(logits)
        if any(math.isnan(l) for l in logits) or m == math.inf:
            s = [math.nan] * E
        else:
            p = [0.0 if l == -math.inf else math.exp(l - m) for l in logits]
            s = [v / sum(p) if sum(p) else 0.0 for v in p]
    c = [a + (bias[e] if bias is not None else 0.0) for e, a in enumerate(s)]
    if any(math.isnan(v) for v in c):
        return list(range(K)), [math.nan] * K
    c = [-math.inf if l == -math.inf else v for l, v in zip(logits, c)]
    n = E // n_group
    if topk_group < n_group:
        best = []
        for g in range(n_group):
            top = sorted(c[g * n:(g + 1) * n], reverse=True)[:group_top]
            top = [v for v in top if v > -math.inf]   # masked experts are no part of a group's sum
            best.append(sum(top) if top else -math.inf)
        open_ = sorted(range(n_group), key=lambda g: (-best[g], g))[:topk_group]
        c = [v if e // n in open_ else -math.inf for e, v in enumerate(c)]
    ids = [e for e in sorted(range(E), key=lambda e: (-c[e], e)) if c[e] > -math.inf][:K]
    w = [s[e] for e in ids]
    if renorm:
        w = [v / sum(w) if sum(w) else 0.0 for v in w]
    left = K - len(ids)
    return ids + [-1] * left, [v * scale for v in w] + [0.0] * left
