"""Products on rows sorted by expert, their gradients, int8 products and the int8 quantizer on the device, against 64-bit
references whose bounds count every rounding (products_ref)."""
import ctypes

import pytest
import torch

import nanovllm_moe
import products_ref as ref
from helpers import topk_routing

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _say(*a):
    print(*a, flush=True)


def _starts(counts, head=0):
    s = [head]
    for c in counts:
        s.append(s[-1] + c)
    return torch.tensor(s, dtype=torch.int32)


def _data(E, N, K, M, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dt)
    w = (torch.randn(E, N, K, generator=g) * 0.1).to(dt)
    dy = torch.randn(M, N, generator=g).to(dt)
    return x, w, dy


def _check_all(cuda, x, w, dy, starts, what=""):
    """Forward and both gradients, through autograd and through the ops."""
    ops, E, dt = torch.ops.nanovllm, w.shape[0], x.dtype
    xc, wc = (t.to(cuda).detach().requires_grad_() for t in (x, w))
    gc, sc = dy.to(cuda), starts.to(cuda)
    _say("[products]", what, tuple(x.shape), tuple(w.shape), dt)
    y = ops.moe_grouped_matmul(xc, wc, sc)
    dx, dw = torch.autograd.grad(y, (xc, wc), gc)
    assert y.dtype == dx.dtype == dw.dtype == dt and dx.shape == x.shape and dw.shape == w.shape
    assert torch.equal(dx, ops.moe_grouped_matmul_dx(gc, wc, sc)) and torch.equal(dw, ops.moe_grouped_matmul_dw(gc, xc, sc))
    st = starts.tolist()
    r = ref.within(y.detach(), *ref.grouped(x, w, st, dt)), ref.within(dx, *ref.grouped_dx(dy, w, st, dt)), \
        ref.within(dw, *ref.grouped_dw(dy, x, st, E, dt))
    assert max(r) <= 1.0, r


# rows of each expert, rows before the first and behind the last
COUNTS = [([1], 0, 0), ([0, 3, 0], 0, 0), ([16, 17, 15, 0], 0, 5), ([33, 64, 1, 65], 3, 0), ([128, 129, 0, 255], 0, 1),
          ([256, 257, 300], 0, 40), ([0, 0, 520, 0], 7, 300), ([0, 0], 0, 9), ([2] * 70, 0, 1)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,head,tail", COUNTS)
@pytest.mark.parametrize("N,K", [(64, 64), (8, 16), (264, 200), (520, 72)])
def test_grouped(cuda, dt, counts, head, tail, N, K):
    E, M = len(counts), head + sum(counts) + tail
    x, w, dy = _data(E, N, K, M, DT[dt], seed=N + K + M)
    _check_all(cuda, x, w, dy, _starts(counts, head))


@pytest.mark.parametrize("N,K", [(1, 1), (7, 64), (64, 7), (257, 129), (33, 1000)])
def test_grouped_odd_sizes(cuda, N, K):
    """Row lengths that are no multiple of 8: the ops copy to padded rows."""
    counts = [5, 0, 40]
    x, w, dy = _data(3, N, K, 48, torch.bfloat16, seed=N * K)
    _check_all(cuda, x, w, dy, _starts(counts))


@pytest.mark.parametrize("N,K,counts", [(768, 2048, [300, 20, 700]), (2048, 1440, [129, 511]), (4096, 4096, [70])])
def test_grouped_long(cuda, N, K, counts):
    x, w, dy = _data(len(counts), N, K, sum(counts), torch.bfloat16, seed=N)
    _check_all(cuda, x, w, dy, _starts(counts))


# Calls of more work than the few-rows kernel takes, one for each tile shape, and with several tiles a workgroup.
# rows of each expert, head, tail, N, K
TILES = {"256x256": ([300] * 8, 0, 7, 4104, 256), "256x128": ([250, 250, 3, 250], 2, 0, 2056, 1032),
         "128x128": ([513], 0, 0, 2048, 1600), "256x64": ([33] * 12, 0, 0, 1280, 2048), "128x64": ([400], 0, 3, 1000, 2056),
         "rounds": ([1000, 3, 900, 1200], 0, 300, 8200, 136), "mixed": ([10, 200, 300, 0, 70, 129, 512, 1] * 5, 5, 270, 4104, 96),
         "one step": ([700, 0, 900], 0, 0, 9000, 64), "long": ([130, 257], 0, 0, 1032, 4104)}


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("name", TILES)
def test_grouped_tiles(cuda, dt, name):
    counts, head, tail, N, K = TILES[name]
    g = torch.Generator(device="cuda").manual_seed(N + K)
    M, E = head + sum(counts) + tail, len(counts)
    x, w, dy = (torch.randn(*s, generator=g, device=cuda).to(DT[dt]) for s in ((M, K), (E, N, K), (M, N)))
    _check_all(cuda, x, w, dy, _starts(counts, head), name)


def test_grouped_many_experts(cuda):
    """512 experts, most without rows; 511 and 513 rows of the first and last."""
    counts = [511] + [0] * 200 + [1, 2, 3] + [0] * 307 + [513]
    x, w, dy = _data(512, 16, 32, sum(counts) + 2, torch.float16, seed=3)
    _check_all(cuda, x, w, dy, _starts(counts))


@pytest.mark.parametrize("starts", [[0, 9, 4, 12], [5, 5, 5, 5], [-3, 4, 8, 100], [100, 100, 100, 100], [12, 3, 20, 0],
                                    [-2 ** 31, 2 ** 31 - 1, 0, 5]])
def test_grouped_any_starts(cuda, starts):
    """starts that do not ascend, or leave [0, M], are read as their running maximum within it."""
    x, w, dy = _data(3, 24, 40, 12, torch.bfloat16, seed=5)
    _check_all(cuda, x, w, dy, torch.tensor(starts, dtype=torch.int32))


def test_grouped_beyond_32_bits(cuda):
    """Weights, rows, outputs and gradients of more than 4 GiB, checked at their ends."""
    ops, dt = torch.ops.nanovllm, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(1)
    E, N, K = 36, 8192, 8192   # 4.8 GB of weights
    w = torch.empty(E, N, K, dtype=dt, device=cuda)
    for e in (0, E - 1):
        w[e] = torch.randn(N, K, generator=g, device=cuda) * 0.02
    s = _starts([70] + [0] * (E - 2) + [90])
    x, dy = (torch.randn(160, n, generator=g, device=cuda).to(dt) for n in (K, N))
    y, dx = ops.moe_grouped_matmul(x, w, s.to(cuda)), ops.moe_grouped_matmul_dx(dy, w, s.to(cuda))
    dw = ops.moe_grouped_matmul_dw(dy, x, s.to(cuda))
    for e, r in ((0, slice(0, 70)), (E - 1, slice(70, 160))):
        st = [0, r.stop - r.start]
        assert ref.within(y[r], *ref.grouped(x[r], w[e:e + 1], st, dt)) <= 1.0
        assert ref.within(dx[r], *ref.grouped_dx(dy[r], w[e:e + 1], st, dt)) <= 1.0
        assert ref.within(dw[e:e + 1], *ref.grouped_dw(dy[r], x[r], st, 1, dt)) <= 1.0
    assert not bool(dw[1:E - 1].any())
    del w, dw, x, dy, y, dx
    M, N, K = 300000, 8192, 64   # 4.9 GB of outputs, then of rows
    x, w = torch.randn(M, K, generator=g, device=cuda).to(dt), torch.randn(2, N, K, generator=g, device=cuda).to(dt)
    s = torch.tensor([0, 100000, M - 3], dtype=torch.int32, device=cuda)
    y = ops.moe_grouped_matmul(x, w, s)
    assert ref.within(y[M - 500:M - 3], *ref.grouped(x[M - 500:M - 3], w[1:], [0, 497], dt)) <= 1.0
    assert ref.within(y[99990:100000], *ref.grouped(x[99990:100000], w[:1], [0, 10], dt)) <= 1.0
    assert not bool(y[M - 3:].any())
    dx = ops.moe_grouped_matmul_dx(y, w, s)
    assert ref.within(dx[M - 500:], *ref.grouped_dx(y[M - 500:], w[1:], [0, 497], dt)) <= 1.0


def test_grouped_one_gradient(cuda):
    """Only x, or only w, with a gradient; outputs of a sum (a gradient with stride 0)."""
    x, w, _ = _data(3, 40, 48, 30, torch.bfloat16, seed=4)
    s = _starts([10, 0, 18])
    one = torch.ones(30, 40, dtype=torch.bfloat16)
    for leaf in ("x", "w"):
        a, b = x.to(cuda), w.to(cuda)
        (a if leaf == "x" else b).requires_grad_()
        torch.ops.nanovllm.moe_grouped_matmul(a, b, s.to(cuda)).sum().backward()
        if leaf == "x":
            assert b.grad is None and ref.within(a.grad, *ref.grouped_dx(one, w, s.tolist(), torch.bfloat16)) <= 1.0
        else:
            assert a.grad is None and ref.within(b.grad, *ref.grouped_dw(one, x, s.tolist(), 3, torch.bfloat16)) <= 1.0


def test_grouped_layouts(cuda):
    """Views: rows of a wider tensor, a slice of the weights' rows, weights stored across, one weight for all experts."""
    E, N, K, counts = 4, 48, 64, [3, 40, 0, 20]
    s = _starts(counts)
    M = sum(counts)
    x, w, dy = _data(E, 2 * N, 2 * K, M, torch.bfloat16, seed=11)
    ops = torch.ops.nanovllm
    cases = {"wide rows": (x[:, K:], w[:, :N, K:], dy[:, N:]), "expert slice": (x[:, :K], w[:, N:, :K], dy[:, :N]),
             "misaligned": (x[:, 1:K + 1], w[:, 1:N + 1, 3:K + 3], dy[:, 5:N + 5]),
             "across": (x[:, :K], w.transpose(1, 2)[:, :K, :N].transpose(1, 2).contiguous().transpose(1, 2), dy[:, :K]),
             "one weight": (x[:, :K], w[:1, :N, :K].expand(E, N, K), dy[:, :N]),
             "row stride": (x[::2], w[::2][:, ::2], dy[::2, :N])}
    for name, (a, b, g) in cases.items():
        b = b.transpose(1, 2) if name == "across" and b.shape[2] != a.shape[1] else b
        big = {}
        for k, t in (("x", a), ("w", b), ("dy", g)):   # the same views on the device
            base = torch.empty(t.untyped_storage().nbytes() // 2, dtype=t.dtype)
            base.copy_(torch.as_strided(t, (base.numel(),), (1,), 0))
            big[k] = torch.as_strided(base.to(cuda), t.shape, t.stride(), t.storage_offset())
        e, m = b.shape[0], a.shape[0]
        st = s if name != "row stride" else torch.tensor([0, 5, m - 2], dtype=torch.int32)
        _say("[products] layout", name, a.stride(), b.stride(), g.stride())
        sc = st.to(cuda)
        y = ops.moe_grouped_matmul(big["x"], big["w"], sc)
        gg = g[:, :b.shape[1]]
        dx = ops.moe_grouped_matmul_dx(big["dy"][:, :b.shape[1]], big["w"], sc)
        dw = ops.moe_grouped_matmul_dw(big["dy"][:, :b.shape[1]], big["x"], sc)
        r = (ref.within(y, *ref.grouped(a, b, st.tolist(), a.dtype)), ref.within(dx, *ref.grouped_dx(gg, b, st.tolist(), a.dtype)),
             ref.within(dw, *ref.grouped_dw(gg, a, st.tolist(), e, a.dtype)))
        assert max(r) <= 1.0, (name, r)


def test_grouped_gradient_of_views(cuda):
    """Gradients through weights stored across and through one weight shared by all experts."""
    E, N, K, counts = 3, 40, 56, [9, 0, 30]
    x, w, dy = _data(E, N, K, sum(counts), torch.float16, seed=2)
    s = _starts(counts)
    ops = torch.ops.nanovllm
    across = w.transpose(1, 2).contiguous().to(cuda).requires_grad_()   # [E,K,N]
    y = ops.moe_grouped_matmul(x.to(cuda), across.transpose(1, 2), s.to(cuda))
    (gw,) = torch.autograd.grad(y, across, dy.to(cuda))
    dw, bound = ref.grouped_dw(dy, x, s.tolist(), E, torch.float16)
    assert ref.within(y.detach(), *ref.grouped(x, w, s.tolist(), torch.float16)) <= 1.0
    assert ref.within(gw.transpose(1, 2), dw, bound) <= 1.0
    one = w[0].to(cuda).requires_grad_()
    y = ops.moe_grouped_matmul(x.to(cuda), one.expand(E, N, K), s.to(cuda))
    (g1,) = torch.autograd.grad(y, one, dy.to(cuda))
    # autograd adds the experts' gradients in 16 bits: E - 1 more roundings of partial sums
    mag = dw.abs().sum(0) + bound.sum(0)
    assert ref.within(g1, dw.sum(0), bound.sum(0) + mag * (E * torch.finfo(torch.float16).eps)) <= 1.0


def test_grouped_gradient_against_differences(cuda):
    """The gradients of a sum of outputs against central differences of the kernel's own forward, which is linear."""
    E, N, K, counts = 2, 16, 24, [5, 11]
    g = torch.Generator().manual_seed(9)
    # multiples of 1/4 up to 1: outputs are multiples of 1/16 up to 24, and up to 56 with one value 32 further
    x = (torch.randint(-4, 5, (16, K), generator=g) / 4).to(torch.bfloat16)
    w = (torch.randint(-4, 5, (E, N, K), generator=g) / 4).to(torch.bfloat16)
    dy = torch.zeros(16, N).to(torch.bfloat16)
    dy[3, 5] = dy[9, 2] = 1.0
    s = _starts(counts).to(cuda)
    ops = torch.ops.nanovllm

    def loss(a, b):
        y = ops.moe_grouped_matmul(a.to(cuda), b.to(cuda), s).float().cpu()
        return float(y[3, 5] + y[9, 2])

    dx = ops.moe_grouped_matmul_dx(dy.to(cuda), w.to(cuda), s).float().cpu()   # exact: single products by 1
    dw = ops.moe_grouped_matmul_dw(dy.to(cuda), x.to(cuda), s).float().cpu()
    # only the outputs' rounding to 8 bits: half a step of 2^-2 below 64, in four outputs, over the distance 64
    tol = 4 * 2.0 ** -3 / 64
    for r, k in ((3, 0), (3, 23), (9, 7), (4, 4)):
        step = torch.zeros_like(x)
        step[r, k] = 32
        d = (loss(x + step, w) - loss(x - step, w)) / 64
        assert abs(d - float(dx[r, k])) <= tol, (r, k, d, float(dx[r, k]))
    for e, n, k in ((0, 5, 1), (1, 2, 20), (0, 2, 3), (1, 5, 0)):
        step = torch.zeros_like(w)
        step[e, n, k] = 32
        d = (loss(x, w + step) - loss(x, w - step)) / 64
        assert abs(d - float(dw[e, n, k])) <= tol, (e, n, k, d, float(dw[e, n, k]))


def test_grouped_neighbours_do_not_leak(cuda):
    """NaN and infinities in rows of no expert, in another expert's rows and in unused experts' weights stay there."""
    counts, N, K = [20, 0, 13], 72, 88
    s = _starts(counts, head=2)
    x, w, dy = _data(3, N, K, 40, torch.bfloat16, seed=8)
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    x2[:2], x2[35:], dy2[:2], dy2[35:] = float("nan"), float("inf"), float("nan"), -float("inf")
    w2[1] = float("nan")
    ops, sc = torch.ops.nanovllm, s.to(cuda)
    for f, a, b in ((ops.moe_grouped_matmul, (x, w), (x2, w2)), (ops.moe_grouped_matmul_dx, (dy, w), (dy2, w2)),
                    (ops.moe_grouped_matmul_dw, (dy, x), (dy2, x2))):
        assert torch.equal(f(a[0].to(cuda), a[1].to(cuda), sc), f(b[0].to(cuda), b[1].to(cuda), sc))
    x2 = x.clone()
    x2[7, 3] = float("nan")   # one row of expert 0: its outputs alone
    y, y2 = ops.moe_grouped_matmul(x.to(cuda), w.to(cuda), sc), ops.moe_grouped_matmul(x2.to(cuda), w.to(cuda), sc)
    keep = torch.arange(40) != 7
    assert bool(y2[7].isnan().all()) and torch.equal(y[keep.to(cuda)], y2[keep.to(cuda)])


def test_grouped_empty_calls(cuda):
    ops = torch.ops.nanovllm
    s = torch.zeros(3, dtype=torch.int32, device=cuda)
    w = torch.ones(2, 24, 16, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    x = torch.empty(0, 16, dtype=torch.bfloat16, device=cuda, requires_grad=True)
    y = ops.moe_grouped_matmul(x, w, s)
    assert y.shape == (0, 24)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w))


def test_grouped_refusals(cuda):
    ops = torch.ops.nanovllm
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device=cuda)
    w = torch.zeros(2, 24, 16, dtype=torch.bfloat16, device=cuda)
    s = torch.zeros(3, dtype=torch.int32, device=cuda)
    f = ops.moe_grouped_matmul
    for call, word in ((lambda: f(x[0], w, s), "expected"), (lambda: f(x, w[0], s), "expected"), (lambda: f(x[:, :8], w, s), "expected"),
                       (lambda: f(x.half(), w, s), "one dtype"), (lambda: f(x.float(), w.float(), s), "float16 or bfloat16"),
                       (lambda: f(x, w, s[:2]), "E="), (lambda: f(x, w, s.long()), "int32"), (lambda: f(x, w, s.cpu()), "same device"),
                       (lambda: f(x, w.cpu(), s), "same device"), (lambda: ops.moe_grouped_matmul_dx(x, w, s), "expected"),
                       (lambda: ops.moe_grouped_matmul_dw(x, x[:3], s), "expected")):
        with pytest.raises(RuntimeError, match=word):
            call()
    x.requires_grad_()
    y = f(x, w, s)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)


# ------------------------------------------------------------------------------------------ int8
def _codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
    return q, torch.rand(shape[:-1], generator=g) * 0.02 + 0.001


OUT = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 96, 2048), (5, 33, 64), (16, 256, 128), (17, 100, 208), (64, 1000, 144),
                                   (65, 64, 1024), (130, 257, 80), (300, 514, 512), (513, 72, 32)])
@pytest.mark.parametrize("bias", [False, True])
def test_int8_matmul(cuda, out, M, N, K, bias):
    x, xs = _codes((M, K), M + K)
    w, ws = _codes((N, K), N)
    xs, ws = xs * 0.05, ws * 0.05   # outputs stay far below fp16's largest
    b = torch.randn(N, generator=torch.Generator().manual_seed(K)) if bias else None
    _say("[int8]", M, N, K, out)
    y = torch.ops.nanovllm.int8_matmul(x.to(cuda), xs.to(cuda), w.to(cuda), ws.to(cuda), None if b is None else b.to(cuda), out)
    assert y.dtype == out
    assert ref.within(y, *ref.int8_rows(x, xs, w, ws, b, out)) <= 1.0


def test_int8_extremes(cuda):
    """The longest sums of the largest codes, exact in int32, from rows that are no whole pieces of 16; NaN scales."""
    K = 131055
    x, w = torch.full((3, K), -128, dtype=torch.int8), torch.full((5, K), -128, dtype=torch.int8)
    x[1], w[2] = 127, 127
    one = torch.ones(5)
    f = torch.ops.nanovllm.int8_matmul
    y = f(x.to(cuda), one[:3].to(cuda), w.to(cuda), one.to(cuda), None, torch.float32)
    assert ref.within(y, *ref.int8_rows(x, one[:3], w, one, None, torch.float32)) <= 1.0
    xs = torch.tensor([1.0, float("nan"), 2.0])
    y = f(x.to(cuda), xs.to(cuda), w.to(cuda), one.to(cuda), None, torch.float32).cpu()
    assert bool(y[1].isnan().all()) and bool(torch.isfinite(y[[0, 2]]).all())
    x, w = torch.full((200, K), -128, dtype=torch.int8, device=cuda), torch.full((300, K), -128, dtype=torch.int8, device=cuda)
    x[::3], w[::2] = 127, 126   # the same sums through tiles
    s = torch.ones(300, device=cuda)
    y = f(x, s[:200], w, s, None, torch.float32)
    assert ref.within(y, *ref.int8_rows(x, s[:200], w, s, None, torch.float32)) <= 1.0
    y = f(x[:1].expand(5, K), s[:5], w, s, None, torch.float32)   # one row for all
    assert ref.within(y, *ref.int8_rows(x[:1].expand(5, K), s[:5], w, s, None, torch.float32)) <= 1.0
    with pytest.raises(RuntimeError, match="int32"):
        big = torch.zeros(1, 131057, dtype=torch.int8, device=cuda)
        f(big, one[:1].to(cuda), big, one[:1].to(cuda), None, torch.float32)


def test_int8_layouts_and_refusals(cuda):
    f = torch.ops.nanovllm.int8_matmul
    x, xs = _codes((40, 160), 1)
    w, ws = _codes((50, 160), 2)
    xc, wc, xsc, wsc = x.to(cuda), w.to(cuda), xs.to(cuda), ws.to(cuda)
    for a, b in ((slice(0, 64), slice(64, 128)), (slice(3, 67), slice(1, 65)), (slice(0, 33), slice(16, 49))):
        y = f(xc[:, a], xsc, wc[:, b], wsc, None, torch.float32)
        assert ref.within(y, *ref.int8_rows(x[:, a], xs, w[:, b], ws, None, torch.float32)) <= 1.0
    y = f(xc[::3], xsc[::3], wc[::2], wsc[::2], None, torch.float32)
    assert ref.within(y, *ref.int8_rows(x[::3], xs[::3], w[::2], ws[::2], None, torch.float32)) <= 1.0
    y = f(xc, xsc, wc.t().contiguous().t(), wsc, None, torch.float32)
    assert ref.within(y, *ref.int8_rows(x, xs, w, ws, None, torch.float32)) <= 1.0
    assert f(xc[:0], xsc[:0], wc, wsc, None, torch.float32).shape == (0, 50)
    for call, word in ((lambda: f(xc.float(), xsc, wc, wsc, None, torch.float32), "int8"),
                       (lambda: f(xc, xsc.half(), wc, wsc, None, torch.float32), "float32"),
                       (lambda: f(xc, xsc[:3], wc, wsc, None, torch.float32), "x_scales"),
                       (lambda: f(xc, xsc, wc, wsc[:3], None, torch.float32), "w_scales"),
                       (lambda: f(xc, xsc, wc[:, :64], wsc, None, torch.float32), "expected"),
                       (lambda: f(xc, xsc, wc, wsc, wsc[:3], torch.float32), "bias"),
                       (lambda: f(xc, xsc, wc, wsc, None, torch.float64), "dtype"),
                       (lambda: f(xc, xsc, wc.cpu(), wsc, None, torch.float32), "same device")):
        with pytest.raises(RuntimeError, match=word):
            call()


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("counts,head,tail", COUNTS)
@pytest.mark.parametrize("N,K", [(72, 64), (7, 16), (300, 208)])
def test_int8_grouped(cuda, out, counts, head, tail, N, K):
    E, M = len(counts), head + sum(counts) + tail
    x, xs = _codes((M, K), M)
    w, ws = _codes((E, N, K), N)
    xs = xs * 0.05
    s = _starts(counts, head)
    _say("[int8 grouped]", counts[:8], N, K, out)
    y = torch.ops.nanovllm.moe_grouped_matmul_int8(x.to(cuda), xs.to(cuda), w.to(cuda), ws.to(cuda), s.to(cuda), out)
    assert ref.within(y, *ref.int8_grouped(x, xs, w, ws, s.tolist(), out)) <= 1.0


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("name", TILES)
def test_int8_tiles(cuda, out, name):
    counts, head, tail, N, K = TILES[name]
    K = 2 * K // 16 * 16
    M, E = head + sum(counts) + tail, len(counts)
    g = torch.Generator(device="cuda").manual_seed(N + K)
    x, w = (torch.randint(-128, 128, s, generator=g, device=cuda, dtype=torch.int32).to(torch.int8) for s in ((M, K), (E, N, K)))
    xs, ws = (torch.rand(s, generator=g, device=cuda) * 0.001 + 1e-5 for s in ((M,), (E, N)))
    s = _starts(counts, head)
    _say("[int8 tiles]", name, M, N, K, E, out)
    ops = torch.ops.nanovllm
    y = ops.moe_grouped_matmul_int8(x, xs, w, ws, s.to(cuda), out)
    assert ref.within(y, *ref.int8_grouped(x, xs, w, ws, s.tolist(), out)) <= 1.0
    bias = torch.randn(N, generator=g, device=cuda)
    y = ops.int8_matmul(x, xs, w[0], ws[0], bias, out)
    assert ref.within(y, *ref.int8_rows(x, xs, w[0], ws[0], bias, out)) <= 1.0


def _same_codes(cuda, x):
    q, s = torch.ops.nanovllm.int8_quantize(x)
    rq, rs = ref.quantize(x.cpu())
    assert torch.equal(s.cpu().isnan(), rs.isnan()) and torch.equal(s.cpu().nan_to_num(0.0), rs.nan_to_num(0.0))
    assert torch.equal(q.cpu(), rq)
    for dt in OUT:
        v = torch.ops.nanovllm.int8_dequantize(q, s, dt)
        r = rq.double() * rs.double().unsqueeze(-1)
        # the product in fp32 (2^-24 of it; the fp16 conversion may take the exact product), then half a step of dt; beyond
        # dt's largest value an infinity
        bad, big = r.isnan(), r.abs() >= torch.finfo(dt).max
        v = v.cpu()
        assert v.dtype == dt and torch.equal(v.isnan(), bad) and bool((v[big].abs() >= torch.finfo(dt).max).all())
        keep = ~(bad | big)
        assert ref.within(v[keep], r[keep], ref.round_bound(r, r.abs() * 2.0 ** -24, dt)[keep]) <= 1.0


@pytest.mark.parametrize("dt", OUT)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 2048), (1100, 512), (1030, 1000), (1025, 2048), (7, 4096), (9, 2056),
                                       (4, 16384), (3, 16392), (2, 40000), (2000, 33), (0, 64)])
def test_quantize(cuda, dt, rows, cols):
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))
    _say("[int8 quantize]", rows, cols, dt)
    _same_codes(cuda, x.to(dt).to(cuda))


def test_quantize_many_rows(cuda):
    """More rows than one launch takes, and more than 2^32 values."""
    ops = torch.ops.nanovllm
    g = torch.Generator(device="cuda").manual_seed(2)
    for rows, cols in (((1 << 23) + 5, 8), (2200000, 2048)):
        x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
        pick = torch.tensor([0, 1, (1 << 21) - 1, 1 << 21, rows // 2, rows - 2, rows - 1], device=cuda)
        if rows > 1 << 23:
            pick = torch.cat([pick, torch.tensor([(1 << 23) - 1, 1 << 23, (1 << 23) + 1], device=cuda)])
        x[pick] = torch.randn(len(pick), cols, generator=g, device=cuda).to(torch.bfloat16)
        q, s = ops.int8_quantize(x)
        rq, rs = ref.quantize(x[pick].cpu())
        assert torch.equal(q[pick].cpu(), rq) and torch.equal(s[pick].cpu(), rs)
        v = ops.int8_dequantize(q, s, torch.float32)[pick].cpu()
        assert torch.equal(v, rq.float() * rs.unsqueeze(1))
        del x, q, s, v


def test_quantize_borders(cuda):
    """Quotients on and next to the borders between codes, tiny and huge rows, zeros, NaN and infinities."""
    k = torch.arange(-127, 127, dtype=torch.float32) + 0.5
    rows = []
    for top in (127.0, 127 * 2.0 ** -20, 127 * 3.0, 100.3, 1.7):
        s = torch.tensor(top / 127.0)
        t = k * s
        rows += [torch.cat([t, torch.tensor([top, 0.0])]), torch.cat([torch.nextafter(t, torch.tensor(1e9)), torch.tensor([top, 0.0])]),
                 torch.cat([torch.nextafter(t, torch.tensor(-1e9)), torch.tensor([top, 0.0])])]
    x = torch.stack(rows)
    more = torch.zeros(12, 256)
    more[0, 3] = 2.0 ** -149
    more[1] = torch.arange(256) * 2.0 ** -149
    more[2] = torch.linspace(-1, 1, 256) * 2.0 ** -120
    more[3] = torch.linspace(-1, 1, 256) * 3.4e38
    more[5, 7] = float("nan")
    more[6, 250] = float("inf")
    more[7, 0] = -float("inf")
    more[8] = torch.linspace(-1, 1, 256) * 2.0 ** -126 * 127
    more[9, 100] = 127 * 2.0 ** -126
    more[10] = -0.0
    _same_codes(cuda, torch.cat([x, more]).to(cuda))
    for dt in (torch.bfloat16, torch.float16):
        _same_codes(cuda, torch.cat([x, more]).clamp(-60000, 60000).to(dt).to(cuda))


def test_quantize_layouts(cuda):
    g = torch.Generator().manual_seed(4)
    big = torch.randn(70, 256, generator=g).to(torch.bfloat16).to(cuda)
    for v in (big[:, 64:192], big[::3, :96], big[:, 4:69], big.t()[:, :64], big[1:, :32].expand(69, 32), big[0],
              big[:, :33].reshape(35, 2, 33).transpose(0, 1), big[3:4], big[:, ::2]):
        _same_codes(cuda, v)
    ops = torch.ops.nanovllm
    q, s = ops.int8_quantize(big)
    for call, word in ((lambda: ops.int8_quantize(big.double()), "float32, bfloat16 or float16"),
                       (lambda: ops.int8_quantize(big[:, :0]), "C > 0"),
                       (lambda: ops.int8_dequantize(q, s[:3], torch.float32), "expected"),
                       (lambda: ops.int8_dequantize(q, s.cpu(), torch.float32), "one device"),
                       (lambda: ops.int8_dequantize(q, s.half(), torch.float32), "float32"),
                       (lambda: ops.int8_dequantize(q, s, torch.float64), "float32, bfloat16 or float16")):
        with pytest.raises(RuntimeError, match=word):
            call()


# ------------------------------------------------------------------------------------------ as they are used together
def _route(ids, E, cuda):
    """mi_moe_route: rows sorted by expert -> (pair of every row, starts)."""
    T, K = ids.shape
    L = nanovllm_moe.capi()
    counts = torch.empty(E, dtype=torch.int32, device=cuda)
    starts = torch.empty(E + 1, dtype=torch.int32, device=cuda)
    tok = torch.empty(T * K, dtype=torch.int32, device=cuda)
    scat = torch.empty(T * K, dtype=torch.int32, device=cuda)
    nanovllm_moe.check(L.mi_moe_route(ids.data_ptr(), T, K, E, counts.data_ptr(), starts.data_ptr(), tok.data_ptr(),
                                      scat.data_ptr(), nanovllm_moe.stream_ptr()))
    return tok, scat, starts


def _layer(x, ids, tw, E, gate_up, down, cuda):
    """Expert layer of the given products: gather, gate and up, SiLU * up, down, weighted sum; pairs without an expert dropped."""
    T, K = ids.shape
    tok, scat, starts = _route(ids, E, cuda)
    order = torch.argsort(torch.where(scat < 0, T * K, scat), stable=True)   # pair of every sorted row, dropped ones last
    rows = x[order // K]
    g, u = gate_up(rows, starts).float().chunk(2, dim=-1)
    h = (torch.nn.functional.silu(g) * u).to(x.dtype)
    out = down(h, starts).float()
    pairs = torch.zeros(T * K, x.shape[1], device=cuda).index_copy(0, order, out)
    return (pairs.reshape(T, K, -1) * tw.unsqueeze(-1)).sum(1), h, rows, starts, order


def test_w8a8_layer(cuda):
    """int8_quantize -> grouped int8 -> SiLU -> int8_quantize -> grouped int8 -> combine against the same layer in 64 bits on
    the dequantized operands, and the shared expert through int8_matmul."""
    E, H, I, T, K = 8, 256, 96, 50, 3
    ops = torch.ops.nanovllm
    g = torch.Generator().manual_seed(1)
    w13, w2 = torch.randn(E, 2 * I, H, generator=g) * 0.05, torch.randn(E, H, I, generator=g) * 0.05
    q13, s13 = ops.int8_quantize(w13.to(cuda))
    q2, s2 = ops.int8_quantize(w2.to(cuda))
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    ids, tw = topk_routing(T, E, K, seed=1)
    ids[3, 1], ids[7] = -1, torch.tensor([-1, -1, -1], dtype=torch.int32)   # dropped pairs, and a token without an expert
    ids, tw = ids.to(cuda), tw.to(cuda)

    def product(q, s):
        return lambda rows, starts: ops.moe_grouped_matmul_int8(*ops.int8_quantize(rows), q, s, starts, torch.bfloat16)

    y, h, rows, starts, order = _layer(x, ids, tw, E, product(q13, s13), product(q2, s2), cuda)
    # each product against 64 bits on what it was given
    xq, xs = (t.cpu() for t in ops.int8_quantize(rows))
    hq, hs = (t.cpu() for t in ops.int8_quantize(h))
    st = starts.tolist()
    gu = product(q13, s13)(rows, starts)
    assert ref.within(gu, *ref.int8_grouped(xq, xs, q13.cpu(), s13.cpu(), st, torch.bfloat16)) <= 1.0
    out = product(q2, s2)(h, starts)
    assert ref.within(out, *ref.int8_grouped(hq, hs, q2.cpu(), s2.cpu(), st, torch.bfloat16)) <= 1.0
    assert bool((y[7] == 0).all()) and bool(torch.isfinite(y).all())
    # the whole layer against unquantized weights: two int8 operands of about 0.5% noise each in two products
    ref_y = torch.zeros(T, H, dtype=torch.float64)
    xd = x.cpu().double()
    for t in range(T):
        for k in range(K):
            e = int(ids[t, k])
            if e >= 0:
                a, b = (w13[e].double() @ xd[t]).chunk(2)
                ref_y[t] += float(tw[t, k]) * (w2[e].double() @ (torch.nn.functional.silu(a) * b))
    rel = (y.cpu().double() - ref_y).norm() / ref_y.norm()
    assert rel < 0.05, rel
    sq, ss = q13[0], s13[0]
    shared = ops.int8_matmul(*ops.int8_quantize(x), sq, ss, None, torch.bfloat16)
    xq, xs = (t.cpu() for t in ops.int8_quantize(x))
    assert ref.within(shared, *ref.int8_rows(xq, xs, sq.cpu(), ss.cpu(), None, torch.bfloat16)) <= 1.0


def test_training_layer(cuda):
    """Router weights, grouped products and their gradients in one backward pass, against autograd in 64 bits."""
    E, H, I, T, K = 6, 128, 64, 70, 2
    g = torch.Generator().manual_seed(3)
    dt = torch.bfloat16
    w13, w2 = (torch.randn(E, 2 * I, H, generator=g) * 0.1).to(dt), (torch.randn(E, H, I, generator=g) * 0.1).to(dt)
    x = torch.randn(T, H, generator=g).to(dt)
    ids, tw = topk_routing(T, E, K, seed=5)
    dy = torch.randn(T, H, generator=g)
    ops = torch.ops.nanovllm
    leaves = [t.to(cuda).requires_grad_() for t in (x, w13, w2)]
    y, *_ = _layer(leaves[0], ids.to(cuda), tw.to(cuda), E, lambda r, s: ops.moe_grouped_matmul(r, leaves[1], s),
                   lambda r, s: ops.moe_grouped_matmul(r, leaves[2], s), cuda)
    got = torch.autograd.grad(y, leaves, dy.to(cuda))
    d = [t.double().requires_grad_() for t in (x, w13, w2)]
    out = torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        a, b = (d[0][t] @ d[1][e].t()).chunk(2, dim=-1)
        out = out.index_add(0, t, ((torch.nn.functional.silu(a) * b) @ d[2][e].t()) * tw[t, k].double().unsqueeze(1))
    want = torch.autograd.grad(out, d, dy.double())
    # stages rounded to bf16 on the way to any of them: gate_up, h, down, and in the backward pass out, down's dx, h, gate_up's
    # dx and dw: 8 of at most 2^-8 of the values each
    for a, b in zip([y, *got], [out.detach(), *want]):
        rel = (a.detach().cpu().double() - b).norm() / b.norm()
        assert rel < 8 * 2.0 ** -8, rel


def test_captured_and_replayed(cuda):
    """Forward, gradients, int8 products and quantizer captured once, replayed with other inputs between eager work."""
    ops = torch.ops.nanovllm
    E, N, K, M = 5, 136, 192, 90
    xs, ws, gs = _data(E, N, K, M, torch.bfloat16, seed=1)
    x, w, dy = xs.to(cuda), ws.to(cuda), gs.to(cuda)
    starts = _starts([20, 0, 41, 3, 20]).to(cuda)
    q, s = ops.int8_quantize(w)

    def step():
        a = ops.int8_quantize(x)
        return (ops.moe_grouped_matmul(x, w, starts), ops.moe_grouped_matmul_dx(dy, w, starts), ops.moe_grouped_matmul_dw(dy, x, starts),
                ops.moe_grouped_matmul_int8(*a, q, s, starts, torch.float32), ops.int8_dequantize(*a, torch.float32))

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        a, _, b = _data(E, N, K, M, torch.bfloat16, seed=10 + i)
        x.copy_(a)
        dy.copy_(b)
        starts.copy_(_starts([[90, 0, 0, 0, 0], [0, 0, 0, 0, 0], [1, 2, 3, 4, 5], [18] * 5][i]))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, want):
            assert torch.equal(u, v)


def test_two_streams(cuda):
    """Calls that overlap on two streams share nothing."""
    ops = torch.ops.nanovllm
    sets = []
    for i in range(2):
        x, w, dy = _data(4, 256, 512, 300, torch.bfloat16, seed=20 + i)
        s = _starts([100, 50, 0, 140 + i])
        sets.append([t.to(cuda) for t in (x, w, dy, s)])
    want = [(ops.moe_grouped_matmul(x, w, s), ops.moe_grouped_matmul_dw(dy, x, s)) for x, w, dy, s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for st, (x, w, dy, s) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append((ops.moe_grouped_matmul(x, w, s), ops.moe_grouped_matmul_dw(dy, x, s)))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_c_abi(cuda):
    """The C entry points with row strides and outputs at odd addresses (2-byte aligned)."""
    L = nanovllm_moe.capi()
    E, N, K, M = 3, 70, 48, 33
    x, w, dy = _data(E, N, K, M, torch.float16, seed=6)
    s = _starts([10, 3, 17])
    xc = torch.zeros(M, 80, dtype=torch.float16, device=cuda)
    xc[:, 16:64] = x.to(cuda)
    wc, sc = w.to(cuda), s.to(cuda)
    buf = torch.full((M * N + 9,), 7.0, dtype=torch.float16, device=cuda)
    P = ctypes.c_void_p
    nanovllm_moe.check(L.mi_moe_grouped_matmul(P(xc.data_ptr() + 32), 80, wc.data_ptr(), N * K, K, sc.data_ptr(), M, N, K, E,
                                               nanovllm_moe.F16, P(buf.data_ptr() + 6), nanovllm_moe.stream_ptr()))
    torch.cuda.synchronize()
    y = buf[3:3 + M * N].reshape(M, N)
    assert ref.within(y, *ref.grouped(x, w, s.tolist(), torch.float16)) <= 1.0
    assert bool((buf[:3] == 7).all()) and bool((buf[3 + M * N:] == 7).all())   # nothing beside the output is written
