"""MXFP4 expert layers and the MX quantizers on the device: the quantizers bit for bit against the plain producers, the
layer against a 64-bit reference whose bound counts every rounding (mx_ref.layer)."""
import pytest
import torch

import mx_ref
import nanovllm_moe
from helpers import topk_routing, zipf_routing
from nanovllm_moe import formats as fmt
from test_mx_formats import FORMATS, _blocks

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ quantizers
def _same(x, f, cuda):
    codes, scales = torch.ops.nanovllm.mx_quantize(x, f)
    rc, rs = fmt.mx_quantize(x.cpu(), f)
    assert torch.equal(scales.cpu(), rs) and torch.equal(codes.cpu(), rc)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        v = torch.ops.nanovllm.mx_dequantize(codes, scales, f, dt)
        r = fmt.mx_dequant(rc, rs, f).to(dt)
        assert v.dtype == dt and torch.equal(v.cpu().isnan(), r.isnan())
        assert torch.equal(v.cpu().nan_to_num(nan=0.0, posinf=1e30, neginf=-1e30),
                           r.nan_to_num(nan=0.0, posinf=1e30, neginf=-1e30))


@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_bit_exact(cuda, f, dt):
    x = _blocks()
    if dt == torch.float16:
        x = x.clamp(-60000, 60000)
    x[40, 5], x[41, 40], x[42, 95] = float("nan"), float("inf"), -float("inf")
    _same(x.to(dt).to(cuda), f, cuda)


@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("shape", [(1, 32), (5, 2048), (257, 32), (3, 7, 64), (1000, 160), (32,), (0, 64)])
def test_quantize_shapes(cuda, f, shape):
    g = torch.Generator().manual_seed(sum(shape))
    _same(torch.randn(*shape, generator=g).to(torch.bfloat16).to(cuda), f, cuda)


@pytest.mark.parametrize("f", FORMATS)
def test_quantize_layouts(cuda, f):
    g = torch.Generator().manual_seed(2)
    big = torch.randn(70, 256, generator=g).to(torch.bfloat16).to(cuda)
    for v in (big[:, 64:192], big[::3, :96], big[:, 4:68], big.t()[:, :64], big[1:, :32].expand(69, 32),
              torch.randn(4097, generator=g).to(cuda)[1:].reshape(64, 64), big[:, :32].reshape(35, 2, 32).transpose(0, 1)):
        _same(v, f, cuda)


def test_dequantize_any_scale(cuda):
    """Scale bytes that the quantizer never writes: 0 (2^-127, subnormal results) to 254."""
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1)
    for f, n in (("mxfp4", 16), ("mxfp6", 24)):
        g = torch.Generator().manual_seed(n)
        codes = torch.randint(0, 256, (256, n), generator=g, dtype=torch.uint8)
        v = torch.ops.nanovllm.mx_dequantize(codes.to(cuda), scales.to(cuda), f, torch.float32).cpu()
        r = mx_ref.dequant(codes, scales, f).float()
        assert torch.equal(v[:255], r[:255]) and bool(v[255].isnan().all())


def test_op_refusals(cuda):
    ops = torch.ops.nanovllm
    x = torch.zeros(4, 64, device=cuda)
    c, s = ops.mx_quantize(x, "mxfp4")
    for call, word in ((lambda: ops.mx_quantize(x, "mxfp8"), "format"),
                       (lambda: ops.mx_quantize(x[:, :40], "mxfp4"), "multiple of 32"),
                       (lambda: ops.mx_quantize(x.double(), "mxfp4"), "float32, bfloat16 or float16"),
                       (lambda: ops.mx_dequantize(c, s, "mxfp6", torch.float32), "belong"),
                       (lambda: ops.mx_dequantize(c[:2], s, "mxfp4", torch.float32), "belong"),
                       (lambda: ops.mx_dequantize(c, s.cpu(), "mxfp4", torch.float32), "one device"),
                       (lambda: ops.mx_dequantize(c, s, "mxfp4", torch.float64), "float32, bfloat16 or float16")):
        with pytest.raises(RuntimeError, match=word):
            call()


# ------------------------------------------------------------------------------------------ layer
def _handle(E, H, I, seed, cuda, std=0.05):
    g = torch.Generator().manual_seed(seed)
    w13, w2 = torch.randn(E, 2 * I, H, generator=g) * std, torch.randn(E, H, I, generator=g) * std
    a, b = fmt.mx_quantize(w13, "mxfp4"), fmt.mx_quantize(w2, "mxfp4")
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    h.store_mxfp4_repack(*[t.to(cuda) for t in (*a, *b)])
    return h, mx_ref.dequant(*a, "mxfp4"), mx_ref.dequant(*b, "mxfp4")


def _check(h, w13, w2, x, ids, tw, cuda):
    y = torch.ops.nanovllm.moe_forward(x.to(cuda), ids.to(cuda), tw.to(cuda), h)
    ref, bound = mx_ref.layer(x.double(), ids, tw.double(), w13, w2, x.dtype)
    r = mx_ref.within(y.cpu(), ref, bound)
    assert r <= 1.0, r
    return y


SHAPES = [  # E, H, I: multiples of 128 and not, one block, one unit
    (4, 64, 32), (3, 128, 96), (8, 192, 160), (5, 512, 256), (16, 320, 416), (1, 128, 128), (8, 2048, 768)]


@pytest.mark.parametrize("E,H,I", SHAPES)
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 64, 65, 200])
def test_layer(cuda, E, H, I, T):
    K = min(E, 3)
    h, w13, w2 = _handle(E, H, I, E * 7 + I, cuda)
    ids, tw = topk_routing(T, E, K, seed=T)
    g = torch.Generator().manual_seed(T + H)
    dt = torch.bfloat16 if (T + E) % 2 else torch.float16
    x = (torch.randn(T, H, generator=g) * torch.exp(torch.randn(H, generator=g))).to(dt)
    _check(h, w13, w2, x, ids, tw, cuda)


@pytest.mark.parametrize("E,H,I", [(1, 65536, 64), (2, 64, 65536), (2, 64, 4096), (2, 64, 4128), (2, 17472, 32)])
@pytest.mark.parametrize("T,K", [(1, 1), (5, 2), (3, 9), (70, 2)])
def test_layer_long_rows(cuda, E, H, I, T, K):
    """The largest rows, and the largest and the next intermediate on either side of the one-launch decode kernel."""
    h, w13, w2 = _handle(E, H, I, H + I, cuda)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, E, (T, K), generator=g, dtype=torch.int32)
    tw = torch.rand(T, K, generator=g)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    _check(h, w13, w2, x, ids, tw, cuda)


@pytest.mark.parametrize("K", [1, 8, 10, 16, 40, 64])
@pytest.mark.parametrize("T", [1, 4, 9])
def test_layer_top_k(cuda, K, T):
    E, H, I = 64, 256, 128
    h, w13, w2 = _handle(E, H, I, K, cuda)
    ids, tw = topk_routing(T, E, K, seed=K + T)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(K)).to(torch.bfloat16)
    _check(h, w13, w2, x, ids, tw, cuda)


@pytest.mark.parametrize("T", [3, 8, 40, 300])
def test_layer_ids(cuda, T):
    """Ids outside [0, E), an expert twice in one token, one expert for all, tokens with nothing."""
    E, H, I, K = 6, 256, 96, 4
    h, w13, w2 = _handle(E, H, I, 1, cuda)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    tw = torch.rand(T, K, generator=g)
    for ids in (torch.randint(-2, E + 2, (T, K), generator=g), torch.full((T, K), 5), torch.full((T, K), -1),
                torch.full((T, K), E), torch.tensor([0, 0, 3, 2 ** 31 - 1]).expand(T, K)):
        ids = ids.to(torch.int32).contiguous()
        ids[T // 2] = -1
        y = _check(h, w13, w2, x, ids, tw, cuda)
        assert bool((y[T // 2] == 0).all())


@pytest.mark.parametrize("T", [1, 6, 70])
def test_layer_not_finite(cuda, T):
    """NaN and infinity in one token's x: its row is NaN, every other row as without them."""
    E, H, I, K = 4, 256, 96, 2
    h, w13, w2 = _handle(E, H, I, 3, cuda)
    ids, tw = topk_routing(T, E, K, seed=1)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    clean = _check(h, w13, w2, x, ids, tw, cuda)
    for v in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[T // 2, 77] = v
        y = torch.ops.nanovllm.moe_forward(z.to(cuda), ids.to(cuda), tw.to(cuda), h)
        assert bool(y[T // 2].isnan().all())
        keep = torch.arange(T) != T // 2
        assert torch.equal(y[keep.to(cuda)], clean[keep.to(cuda)])
    z = torch.zeros_like(x)
    assert bool((torch.ops.nanovllm.moe_forward(z.to(cuda), ids.to(cuda), tw.to(cuda), h) == 0).all())


def test_layer_skewed_and_prefill(cuda):
    E, H, I, K = 16, 512, 352, 4
    h, w13, w2 = _handle(E, H, I, 9, cuda)
    for T in (129, 700, 1500):
        for routing in (topk_routing, zipf_routing):
            ids, tw = routing(T, E, K, seed=T)
            x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
            _check(h, w13, w2, x, ids, tw, cuda)


def test_online_quantization(cuda):
    """quantize_and_store_expert: the layer of the same weights stored as codes, bit for bit."""
    E, H, I, T, K = 3, 192, 96, 7, 2
    g = torch.Generator().manual_seed(4)
    gate, up, down = (torch.randn(E, *s, generator=g) * 0.05 for s in ((I, H), (I, H), (H, I)))
    ids, tw = topk_routing(T, E, K, seed=4)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        a = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
        b = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
        w13 = torch.cat([gate, up], 1).to(dt)
        a.store_mxfp4_repack(*fmt.mx_quantize(w13, "mxfp4"), *fmt.mx_quantize(down.to(dt), "mxfp4"))   # host tensors
        for e in range(E):
            for name, w in (("gate_proj", gate), ("up_proj", up), ("down_proj", down)):
                v = w[e].to(dt)
                b.quantize_and_store_expert(e, name, v if e == 1 else v.to(cuda))
        y = [torch.ops.nanovllm.moe_forward(x, ids.to(cuda), tw.to(cuda), h) for h in (a, b)]
        assert torch.equal(*y) and float(y[0].abs().max()) > 0


def test_layer_forms_agree(cuda):
    """moe_forward_out, the graph-context op, the call without allocation and repeated calls: the same bits."""
    import ctypes
    E, H, I, K = 16, 256, 192, 4
    h, _, _ = _handle(E, H, I, 5, cuda)
    L = nanovllm_moe.capi()
    hp = ctypes.c_void_p()
    g = torch.Generator().manual_seed(5)
    nanovllm_moe.check(L.mi_moe_create(E, H, I, 3, ctypes.byref(hp)))
    w = [t.to(cuda) for s in ((E, 2 * I, H), (E, H, I)) for t in fmt.mx_quantize(torch.randn(*s, generator=g) * 0.05, "mxfp4")]
    nanovllm_moe.check(L.mi_moe_store_mxfp4(hp, *[t.data_ptr() for t in w], 1, nanovllm_moe.stream_ptr()))
    h.store_mxfp4_repack(*w)
    for T in (1, 8, 30, 100):
        ids, tw = (t.to(cuda) for t in topk_routing(T, E, K, seed=T))
        x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
        y = torch.ops.nanovllm.moe_forward(x, ids, tw, h)
        out = torch.full_like(x, float("nan"))
        torch.ops.nanovllm.moe_forward_out(x, ids, tw, h, out)
        assert torch.equal(y, out)
        ctx = torch.classes.nanovllm.MoEGraphContext(h, T, K, 1)
        torch.ops.nanovllm.moe_forward_npu_graph_out(x, ids, tw, h, ctx, out.fill_(float("nan")))
        assert torch.equal(y, out)
        out.fill_(float("nan"))
        nanovllm_moe.check(L.mi_moe_forward_noalloc(hp, x.data_ptr(), out.data_ptr(), tw.data_ptr(), ids.data_ptr(), T, K,
                                                    nanovllm_moe.BF16, nanovllm_moe.stream_ptr()))
        assert torch.equal(y, out)
    L.mi_moe_destroy(hp)


@pytest.mark.parametrize("T", [1, 8, 70])
def test_layer_graph(cuda, T):
    """Replays with new inputs, eager calls of other sizes between them."""
    E, H, I, K = 16, 512, 256, 8
    h, _, _ = _handle(E, H, I, 6, cuda)
    ids, tw = (t.to(cuda) for t in topk_routing(T, E, K, seed=T))
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    y = torch.empty_like(x)
    ctx = torch.classes.nanovllm.MoEGraphContext(h, T, K, 1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        torch.ops.nanovllm.moe_forward_npu_graph_out(x, ids, tw, h, ctx, y)
    for i in range(4):
        x.copy_(torch.randn(T, H, generator=g).to(torch.bfloat16))
        ids.copy_(topk_routing(T, E, K, seed=100 * i + T)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, torch.ops.nanovllm.moe_forward(x, ids, tw, h))
        big = torch.randn(300 + 200 * i, H, generator=g).to(torch.bfloat16).to(cuda)
        bi, bw = (t.to(cuda) for t in topk_routing(len(big), E, K, seed=i))
        torch.ops.nanovllm.moe_forward(big, bi, bw, h)


@pytest.mark.parametrize("T", [1, 8, 70])
def test_ops_in_a_graph(cuda, T):
    """Router, layer and quantizers captured once, replayed over new inputs: as called eagerly."""
    E, H, I, K = 16, 512, 256, 8
    h, _, _ = _handle(E, H, I, 14, cuda)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
    logits = torch.randn(T, E, generator=g).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.1).to(cuda)
    ops = torch.ops.nanovllm

    def run():
        args = (K, bias, "sigmoid", 4, 2, 2, True, 2.5)
        y = ops.moe_forward_scores(x, logits, *args, h)
        codes, scales = ops.mx_quantize(y, "mxfp6")
        return y, *ops.moe_topk_scores(logits, *args), codes, scales, ops.mx_dequantize(codes, scales, "mxfp6", torch.bfloat16)

    run()   # the handle's buffers
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        x.copy_(torch.randn(T, H, generator=g).to(torch.bfloat16))
        logits.copy_(torch.randn(T, E, generator=g))
        logits[0, i:i + 9] = -float("inf")
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, run()))
        n = 200 * (i + 1)   # an eager call that outgrows the buffers
        ops.moe_forward_scores(x[:1].expand(n, H), logits[:1].expand(n, E), K, None, "softmax", 1, 1, 1, True, 1.0, h)


def test_layer_other_stream(cuda):
    E, H, I, K, T = 8, 256, 128, 4, 33
    h, _, _ = _handle(E, H, I, 7, cuda)
    ids, tw = (t.to(cuda) for t in topk_routing(T, E, K, seed=7))
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(cuda)
    y = torch.ops.nanovllm.moe_forward(x, ids, tw, h)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = torch.ops.nanovllm.moe_forward(x, ids, tw, h)
        q = torch.ops.nanovllm.mx_dequantize(*torch.ops.nanovllm.mx_quantize(x, "mxfp6"), "mxfp6", torch.bfloat16)
    s.synchronize()
    assert torch.equal(y, z)
    assert torch.equal(q.cpu().float(), fmt.mx_dequant(*fmt.mx_quantize(x.cpu(), "mxfp6"), "mxfp6"))


def test_two_handles_at_once(cuda):
    """Decode and sorted calls of two layers on two streams, queued without waiting: each as alone."""
    E, H, I, K = 16, 512, 256, 4
    hs = [_handle(E, H, I, s, cuda)[0] for s in (11, 12)]
    streams = [torch.cuda.Stream() for _ in hs]
    g = torch.Generator().manual_seed(8)
    calls = []
    for T in (1, 8, 16, 100, 400):
        ids, tw = (t.to(cuda) for t in topk_routing(T, E, K, seed=T))
        x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(cuda)
        calls.append((x, ids, tw, [torch.ops.nanovllm.moe_forward(x, ids, tw, h) for h in hs]))
    torch.cuda.synchronize()
    got = []
    for rep in range(6):
        for x, ids, tw, _ in calls:
            for h, s in zip(hs, streams):
                with torch.cuda.stream(s):
                    got.append(torch.ops.nanovllm.moe_forward(x, ids, tw, h))
    torch.cuda.synchronize()
    want = [y for _ in range(6) for c in calls for y in c[3]]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_timing(cuda):
    E, H, I = 8, 256, 128
    h, _, _ = _handle(E, H, I, 13, cuda)
    assert h.get_last_run_time_ms() < 0
    h.set_timing(True)
    for T, K, phases in ((2, 4, 1), (2, 8, 1), (100, 4, 2)):   # one launch; sorted
        ids, tw = (t.to(cuda) for t in topk_routing(T, E, K, seed=T))
        torch.ops.nanovllm.moe_forward(torch.zeros(T, H, dtype=torch.bfloat16, device=cuda), ids, tw, h)
        ms = h.get_last_phase_times_ms()
        assert len(ms) == phases and all(v > 0 for v in ms) and h.get_last_run_time_ms() > 0


def test_layer_refusals(cuda):
    E, H, I, K = 4, 128, 64, 2
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    assert h.get_quant_type() == "MXFP4"
    x = torch.zeros(2, H, dtype=torch.bfloat16, device=cuda)
    ids, tw = (t.to(cuda) for t in topk_routing(2, E, K, seed=0))
    with pytest.raises(RuntimeError, match="not stored"):
        torch.ops.nanovllm.moe_forward(x, ids, tw, h)
    w13, w2 = torch.randn(E, 2 * I, H), torch.randn(E, H, I)
    a, b = fmt.mx_quantize(w13, "mxfp4"), fmt.mx_quantize(w2, "mxfp4")
    for bad, word in (((a[0][:3], a[1], *b), "gate_up"), ((*a, b[0], b[1][..., :1]), "down"),
                      ((a[0].to(cuda), a[1], *b), "one device"), ((a[0].to(torch.int16), a[1], *b), "uint8")):
        with pytest.raises(RuntimeError, match=word):
            h.store_mxfp4_repack(*bad)
    with pytest.raises(RuntimeError, match="W4A16"):
        h.store_awq_repack(*[torch.zeros(1)] * 6, 128)
    with pytest.raises(RuntimeError, match="MXFP4 handle"):
        torch.classes.nanovllm.MoEInfer(E, H, I, 1).store_mxfp4_repack(*a, *b)
    h.store_mxfp4_repack(*a, *b)
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        torch.ops.nanovllm.moe_forward(x.float(), ids, tw, h)
    f, lg = torch.ops.nanovllm.moe_forward_scores, torch.zeros(2, E, device=cuda)
    for args, word in (((x, lg[:1], 2), "T,H"), ((x, lg[:, :3], 2), "experts"), ((x[:, :64], lg, 2), "hidden size"),
                       ((x, lg, 5), "top_k"), ((x, lg.cpu(), 2), "one device"), ((x.float(), lg, 2), "float16 or bfloat16")):
        with pytest.raises(RuntimeError, match=word):
            f(*args, None, "softmax", 1, 1, 1, True, 1.0, h)
    with pytest.raises(RuntimeError, match="one device"):
        f(x, lg, 2, torch.zeros(E), "softmax", 1, 1, 1, True, 1.0, h)
    with pytest.raises(RuntimeError, match="one device"):
        torch.ops.nanovllm.moe_topk_scores(lg.cpu(), 2, torch.zeros(E, device=cuda))
    assert f(x[:0], lg[:0], 2, None, "softmax", 1, 1, 1, True, 1.0, h).shape == (0, H)
    assert torch.ops.nanovllm.moe_forward(x[:0], ids[:0], tw[:0], h).shape == (0, H)
    with pytest.raises(RuntimeError, match="HIP tensors only"):
        torch.ops.nanovllm.moe_forward(x.cpu(), ids.cpu(), tw.cpu(), h)


# ------------------------------------------------------------------------------------------ used together
@pytest.mark.parametrize("T", [1, 3, 8, 50, 260])
def test_router_and_layer(cuda, T):
    """Weights quantized by mx_quantize, hidden states routed by scores and run through the layer, as a model does it."""
    E, H, I, K = 32, 256, 160, 6
    g = torch.Generator().manual_seed(T)
    w13, w2 = (torch.randn(*s, generator=g).to(torch.bfloat16) * 0.05 for s in ((E, 2 * I, H), (E, H, I)))
    a, b = (torch.ops.nanovllm.mx_quantize(w.to(cuda), "mxfp4") for w in (w13, w2))
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    h.store_mxfp4_repack(*a, *b)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    logits, bias = torch.randn(T, E, generator=g), torch.randn(E, generator=g) * 0.1
    logits[T // 2, 3:] = -float("inf")      # three experts left: ids of -1 behind them
    args = (K, bias.to(cuda), "sigmoid", 8, 4, 2, True, 2.5)
    y = torch.ops.nanovllm.moe_forward_scores(x.to(cuda), logits.to(cuda), *args, h)
    ids, tw = torch.ops.nanovllm.moe_topk_scores(logits.to(cuda), *args)
    assert torch.equal(y, torch.ops.nanovllm.moe_forward(x.to(cuda), ids, tw, h))
    assert ids[T // 2, 3:].tolist() == [-1, -1, -1]
    ref, bound = mx_ref.layer(x.double(), ids.cpu(), tw.cpu().double(), *(mx_ref.dequant(*(t.cpu() for t in p), "mxfp4") for p in (a, b)), x.dtype)
    assert mx_ref.within(y.cpu(), ref, bound) <= 1.0
    logits[T // 2, 5] = float("nan")
    y2 = torch.ops.nanovllm.moe_forward_scores(x.to(cuda), logits.to(cuda), *args, h)
    assert bool(y2[T // 2].isnan().all())
    y3 = torch.ops.nanovllm.moe_forward_logits(x.to(cuda), logits.nan_to_num(nan=0.0).to(cuda), K, True, h)
    i3, w3 = torch.ops.nanovllm.moe_topk_softmax(logits.nan_to_num(nan=0.0).to(cuda), K, True)
    assert torch.equal(y3, torch.ops.nanovllm.moe_forward(x.to(cuda), i3, w3, h))
