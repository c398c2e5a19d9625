"""Score router on host and device (moe_topk_scores) against a plain 64-bit one: ids equal, weights within one fp32
rounding (half a step, 2^-24, and 2^-40 for the 64-bit sums)."""
import ctypes
import itertools

import pytest
import torch

import nanovllm_moe
import score_ref

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def dev(request):
    if request.param == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")
    nanovllm_moe.load()
    return torch.device(request.param)


def _check(logits, bias, K, score, groups, top, group_top, renorm, scale, dev):
    ids, w = torch.ops.nanovllm.moe_topk_scores(logits.to(dev), K, None if bias is None else bias.to(dev), score, groups,
                                                top, group_top, renorm, scale)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (len(logits), K)
    b = None if bias is None else bias.tolist()
    sc = torch.tensor(scale, dtype=torch.float32).item()
    ref = [score_ref.route(l, b, K, score == "sigmoid", groups, top, group_top, renorm, sc) for l in logits.double().tolist()]
    assert ids.tolist() == [r[0] for r in ref]
    rw = torch.tensor([r[1] for r in ref], dtype=torch.float64).reshape(w.shape)
    w = w.cpu().double()
    assert torch.equal(w.isnan(), rw.isnan())
    off = ((w - rw).abs() - rw.abs() * (2.0 ** -24 + 2.0 ** -40)).nan_to_num(0.0)
    assert bool((off <= 2.0 ** -150).all()), float(off.max())   # below fp32's normal numbers: half its smallest step


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K,groups,top", [(1, 256, 8, 8, 4), (5, 60, 6, 1, 1), (33, 128, 8, 1, 1), (3, 512, 64, 64, 9),
                                              (7, 96, 12, 3, 2), (2, 1, 1, 1, 1), (130, 16, 2, 8, 1), (4, 511, 3, 7, 7),
                                              (1, 65, 10, 5, 1)])
def test_scores(dev, dt, score, T, E, K, groups, top):
    g = torch.Generator().manual_seed(T * E + K)
    for i, (with_bias, renorm) in enumerate(itertools.product((True, False), (True, False))):
        logits = (torch.randn(T, E, generator=g) * 2).to(dt)
        bias = torch.randn(E, generator=g) * 0.3 if with_bias else None
        group_top = min(1 + i % 2, E // groups)
        _check(logits, bias, K, score, groups, top, group_top, renorm, (1.0, 2.5)[i % 2], dev)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top", [(1, 1), (8, 3), (16, 2)])
def test_ties_and_masks(dev, score, groups, top):
    E, K = 64, 4
    inf, lowest = float("inf"), torch.finfo(torch.float32).min
    x = torch.zeros(14, E)
    x[1] = torch.arange(E).float() % 3            # many ties
    x[2] = -inf                                   # nothing left
    x[3] = -inf
    x[3, 41] = 0.5                                # one expert left
    x[4] = -inf
    x[4, [3, 20, 21]] = torch.tensor([1.0, 0.0, 0.0])
    x[5] = lowest                                 # a mask of the type's lowest value is a score like any other
    x[6] = lowest
    x[6, 17] = 0.0
    x[7, 9] = float("nan")
    x[8, 9] = inf
    x[9] = -1000.0                                # sigmoid scores of 0: the sum of the picks is 0
    x[10] = 1000.0
    x[11, ::2] = -inf
    x[12] = torch.linspace(-40, 40, E)
    x[13, :32] = 7.0
    for bias in (None, torch.zeros(E), (torch.arange(E).float() - 20) * 1e-3):
        for group_top, renorm in itertools.product((1, 2), (True, False)):
            _check(x, bias, K, score, groups, top, group_top, renorm, 1.0, dev)
    b = torch.zeros(E)
    b[5], b[6], b[7] = inf, -inf, -5.0            # always, never, last
    _check(x, b, K, score, groups, top, 2, True, 1.0, dev)
    b[8] = float("nan")
    _check(x, b, K, score, groups, top, 1, True, 1.0, dev)


def test_near_scores(dev):
    """Choices that differ by less than fp32 holds are still told apart: the bias makes up for the score up to 1e-9."""
    E = 128
    l = torch.linspace(-2, 2, E)
    s = 1 / (1 + torch.exp(-l.double()))
    _check(torch.stack([l, l.flip(0)]), (0.9 - s).float(), 8, "sigmoid", 4, 2, 2, True, 1.0, dev)


def test_layouts_and_empty(dev):
    g = torch.Generator().manual_seed(1)
    big = torch.randn(40, 300, generator=g).to(dev)
    for v in (big[:, 7:71], big[::3, :64], big.t()[:64, :40]):
        bias = torch.randn(2 * v.shape[1], generator=g).to(dev)[::2]
        a = torch.ops.nanovllm.moe_topk_scores(v, 5, bias, "sigmoid", 2, 1, 2, True, 1.0)
        b = torch.ops.nanovllm.moe_topk_scores(v.contiguous(), 5, bias.contiguous(), "sigmoid", 2, 1, 2, True, 1.0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ids, w = torch.ops.nanovllm.moe_topk_scores(big[:0], 5)
    assert ids.shape == w.shape == (0, 5)


def test_refusals(dev):
    x, b = torch.zeros(2, 64, device=dev), torch.zeros(64, device=dev)
    f = torch.ops.nanovllm.moe_topk_scores
    for args, word in (((x, 0), "top_k"), ((x, 65), "top_k"), ((x, 9, b, "tanh"), "score must be"),
                       ((x, 4, b, "sigmoid", 3), "n_group"), ((x, 4, b, "sigmoid", 0), "n_group"),
                       ((x, 4, b, "sigmoid", 8, 9), "topk_group"), ((x, 4, b, "sigmoid", 8, 0), "topk_group"),
                       ((x, 4, b, "sigmoid", 8, 2, 3), "group_top"), ((x, 1, b, "sigmoid", 64, 2, 2), "group_top"),
                       ((x, 17, b, "sigmoid", 8, 2), "top_k"), ((x[0], 4), "T,E"), ((x, 4, b[:63]), "bias"),
                       ((x, 4, b.double()), "bias"), ((x.double(), 4), "float32, bfloat16 or float16"),
                       ((torch.zeros(2, 520, device=dev), 4), "E must be")):
        with pytest.raises(RuntimeError, match=word):
            f(*args)


def test_c_refusals():
    L = nanovllm_moe.capi()
    P = ctypes.c_void_p(4096)   # never read
    ok = (2, 2, 64, 4, P, 1, 8, 4, 2, 1, 1.0, P, P, None)

    def call(i, v):
        a = list(ok)
        a[i] = v
        return L.mi_moe_topk_scores(P, *a), L.mi_moe_last_error().decode()
    for i, v, word in ((0, 3, "dtype"), (1, -1, "T must"), (1, (1 << 24) + 1, "T must"), (2, 0, "E must"), (3, 0, "top_k"),
                       (5, 2, "score"), (6, 5, "n_group"), (7, 9, "topk_group"), (8, 0, "group_top"), (11, None, "null")):
        rc, msg = call(i, v)
        assert rc == 1 and word in msg, (i, rc, msg)
    assert call(1, 0)[0] == 0
    rc = L.mi_moe_forward_scores(None, P, P, P, 2, 1, 4, None, 1, 1, 1, 1, 1, 1.0, 1, None, None, None)
    assert rc == 1 and "null handle" in L.mi_moe_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("E,K,groups", [(64, 6, (1, 1, 1)), (60, 16, (1, 1, 1)), (128, 8, (16, 4, 2)), (128, 12, (8, 8, 1)),
                                        (256, 8, (8, 4, 2)), (160, 6, (10, 3, 1)), (240, 1, (15, 2, 2)), (16, 4, (4, 2, 2)),
                                        (256, 20, (8, 4, 2)), (250, 5, (1, 1, 1))])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_many_tokens(E, K, groups, dt):
    """A call of many tokens gives each the bits of a call of few, from unaligned rows as well."""
    nanovllm_moe.load()
    T, f, inf = 4001, torch.ops.nanovllm.moe_topk_scores, float("inf")
    g = torch.Generator().manual_seed(E + K)
    flat = (torch.randn(T * E + 1, generator=g) * 2).to(dt)
    x = flat[:T * E].view(T, E)
    x[5], x[6, 3:], x[7, ::2], x[8, 1] = -inf, -inf, -inf, float("nan")
    x[9], x[10], x[11] = 0.0, torch.finfo(dt).min, x[11].round()     # ties
    x[12, 2], x[3999, 1], x[4000, -1] = inf, -inf, float("nan")
    x[20:400] = x[20:400].round()
    flat = flat.cuda()
    x = flat[:T * E].view(T, E)
    bias = (torch.randn(E + 1, generator=g) * 0.1).cuda()
    for score in ("softmax", "sigmoid"):
        for b in (None, bias[:E]):
            args = (b, score, *groups, True, 2.5)
            ids, w = f(x, K, *args)
            parts = [f(x[i:i + 500], K, *args) for i in range(0, T, 500)]
            assert torch.equal(ids, torch.cat([p[0] for p in parts]))
            assert torch.equal(w.nan_to_num(nan=-1.0), torch.cat([p[1] for p in parts]).nan_to_num(nan=-1.0))
            hi, hw = f(x[:600].cpu(), K, None if b is None else b.cpu(), score, *groups, True, 2.5)
            assert torch.equal(ids[:600].cpu(), hi) and torch.equal(w[:600].cpu().isnan(), hw.isnan())
    y, b = flat[1:].view(T, E), bias[1:]
    for p, q in zip(f(y, K, b, "sigmoid", *groups, False, 1.0), f(y.clone(), K, b.clone(), "sigmoid", *groups, False, 1.0)):
        assert torch.equal(p.nan_to_num(nan=-1.0), q.nan_to_num(nan=-1.0))


def test_forward_scores_on_host(monkeypatch):
    """The host layer behind the host router: as its two steps."""
    monkeypatch.setenv("MIMOE_HOST_WEIGHTS", "1")
    nanovllm_moe.load()
    from nanovllm_moe import formats as fmt
    E, H, I, K, T = 8, 64, 64, 2, 3
    g = torch.Generator().manual_seed(0)
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 1)
    h.store_quantized_repack(*fmt.q4_0_random((E, 2 * I), H, generator=g), *fmt.q4_0_random((E, H), I, generator=g))
    x, logits = torch.randn(T, H, generator=g).to(torch.bfloat16), torch.randn(T, E, generator=g)
    args = (K, torch.randn(E, generator=g), "sigmoid", 4, 2, 2, True, 2.5)
    y = torch.ops.nanovllm.moe_forward_scores(x, logits, *args, h)
    ids, w = torch.ops.nanovllm.moe_topk_scores(logits, *args)
    assert torch.equal(y, torch.ops.nanovllm.moe_forward(x, ids, w, h))
