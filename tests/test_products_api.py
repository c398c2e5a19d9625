"""Products on rows sorted by expert and the int8 quantizer without a GPU: refusals of the C ABI, the registered ops, and
the definition of the quantizer."""
import pytest
import torch

import nanovllm_moe
import products_ref as ref

F16, BF16, F32 = nanovllm_moe.F16, nanovllm_moe.BF16, nanovllm_moe.F32
A = 1 << 20   # an aligned address that no refused call reads


def _refused(rc, word, code=1):
    assert rc == code, rc
    assert word in nanovllm_moe.capi().mi_moe_last_error().decode(), nanovllm_moe.capi().mi_moe_last_error()


def _mm(x=A, xs=64, w=A, we=64 * 64, ws=64, starts=A, M=4, N=64, K=64, E=2, dt=BF16, y=A, fn="mi_moe_grouped_matmul"):
    return getattr(nanovllm_moe.capi(), fn)(x, xs, w, we, ws, starts, M, N, K, E, dt, y, None)


@pytest.mark.parametrize("fn", ["mi_moe_grouped_matmul", "mi_moe_grouped_matmul_dx"])
def test_grouped_refusals(fn):
    for kw, word in ((dict(M=-1), "rows"), (dict(M=(1 << 26) + 1), "rows"), (dict(N=0), "N="), (dict(K=0), "K="),
                     (dict(N=(1 << 20) + 8), "N="), (dict(E=0), "experts"), (dict(E=513), "experts"), (dict(dt=F32), "dtype"),
                     (dict(x=None), "null"), (dict(w=None), "null"), (dict(starts=None), "null"), (dict(y=None), "null"),
                     (dict(x=A + 8), "16-byte"), (dict(w=A + 2), "16-byte"), (dict(xs=68), "16-byte"),
                     (dict(xs=56), "row stride"), (dict(ws=56), "row stride"), (dict(xs=(1 << 22) + 8), "row stride"),
                     (dict(we=-8), "expert stride"), (dict(we=4), "expert stride")):
        _refused(_mm(fn=fn, **kw), word)
    _refused(_mm(fn=fn, N=60, K=60, xs=64), "16-byte")   # a row length that is no whole number of pieces
    _refused(_mm(fn=fn, M=1 << 26, N=1 << 20), "tiles", code=3)
    assert _mm(fn=fn, M=0, x=None, w=None, y=None, starts=None) == 0


def test_dw_refusals():
    L = nanovllm_moe.capi()

    def dw(dy=A, ds=64, x=A, xs=64, starts=A, M=4, N=64, K=64, E=2, dt=BF16, out=A):
        return L.mi_moe_grouped_matmul_dw(dy, ds, x, xs, starts, M, N, K, E, dt, out, None)

    for kw, word in ((dict(M=-1), "rows"), (dict(dt=F32), "dtype"), (dict(dy=None), "null"), (dict(x=None), "null"),
                     (dict(starts=None), "null"), (dict(out=None), "null"), (dict(dy=A + 4), "16-byte"), (dict(N=60), "16-byte"),
                     (dict(K=60), "16-byte"), (dict(ds=56), "row stride"), (dict(starts=None, M=0), "null")):
        _refused(dw(**kw), word)
    _refused(dw(N=1 << 20, K=1 << 20, ds=1 << 20, xs=1 << 20), "tiles", code=3)


def test_int8_refusals():
    L = nanovllm_moe.capi()

    def dense(x=A, xst=64, xs=A, w=A, wst=64, ws=A, bias=None, M=4, N=60, K=64, dt=BF16, y=A):
        return L.mi_moe_int8_matmul(x, xst, xs, w, wst, ws, bias, M, N, K, dt, y, None)

    def grouped(x=A, xst=64, xs=A, w=A, we=64 * 60, wst=64, ws=A, starts=A, M=4, N=60, K=64, E=2, dt=BF16, y=A):
        return L.mi_moe_grouped_matmul_int8(x, xst, xs, w, we, wst, ws, starts, M, N, K, E, dt, y, None)

    for f in (dense, grouped):
        for kw, word in ((dict(M=-1), "rows"), (dict(K=131072, xst=131072, wst=131072), "int32"), (dict(dt=3), "values"),
                         (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"),
                         (dict(y=None), "null"), (dict(K=56), "16-byte"), (dict(xst=72), "16-byte"), (dict(wst=48), "row stride")):
            _refused(f(**kw), word)
        assert f(M=0, x=None, y=None) == 0
    _refused(grouped(starts=None), "null")
    _refused(grouped(E=600), "experts")
    _refused(grouped(we=8), "expert stride")


def test_quantizer_refusals():
    L = nanovllm_moe.capi()
    _refused(L.mi_moe_int8_quantize(A, 3, 4, 64, 64, A, A, None), "values")
    _refused(L.mi_moe_int8_quantize(A, BF16, 4, 0, 64, A, A, None), "cols")
    _refused(L.mi_moe_int8_quantize(A, BF16, -1, 64, 64, A, A, None), "rows")
    _refused(L.mi_moe_int8_quantize(A, BF16, 1 << 30, 1 << 20, 1 << 20, A, A, None), "2^40")
    _refused(L.mi_moe_int8_quantize(A, BF16, 4, 64, 63, A, A, None), "row_stride")
    _refused(L.mi_moe_int8_quantize(None, BF16, 4, 64, 64, A, A, None), "null")
    _refused(L.mi_moe_int8_dequantize(A, None, 4, 64, A, BF16, None), "null")
    _refused(L.mi_moe_int8_dequantize(A, A, 4, 64, A, 3, None), "values")
    assert L.mi_moe_int8_quantize(None, BF16, 0, 64, 64, None, None, None) == 0
    assert L.mi_moe_int8_dequantize(None, None, 0, 64, None, BF16, None) == 0


def test_registered_ops():
    nanovllm_moe.load()
    ops = torch.ops.nanovllm
    assert "(Tensor x, Tensor w, Tensor starts) -> Tensor" in str(ops.moe_grouped_matmul.default._schema)
    assert "(Tensor x) -> (Tensor, Tensor)" in str(ops.int8_quantize.default._schema)
    x, w, s = torch.zeros(2, 16), torch.zeros(1, 16, 16), torch.tensor([0, 2], dtype=torch.int32)
    for call in (lambda: ops.moe_grouped_matmul(x, w, s), lambda: ops.int8_quantize(x),
                 lambda: ops.int8_matmul(x, x[:, 0], w[0], w[0, :, 0], None, torch.float32)):
        with pytest.raises((RuntimeError, NotImplementedError), match="CPU"):   # HIP tensors only
            call()


def test_quantizer_definition():
    """The reference's codes are the nearest: no other code is nearer, and a tie is even."""
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(60, 50, generator=g) * torch.exp2(torch.arange(60.0) * 4 - 140).unsqueeze(1),
                   torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5] + [0.0] * 44])])
    q, s = ref.quantize(x)
    assert int(q[60, 1]) == 0 and int(q[60, 2]) == 2 and int(q[60, 3]) == 2 and int(q[60, 5]) == -2
    err = (x.double() - q.double() * s.double().unsqueeze(1)).abs()
    assert bool((err <= s.double().unsqueeze(1) / 2).all())
    assert bool((q.abs().amax(1) <= 127).all())
