"""The MX formats' plain producers (nanovllm_moe.formats) against a 64-bit grid search, and the refusals of the MX
entry points, which need no device."""
import ctypes

import pytest
import torch

import mx_ref
import nanovllm_moe
from nanovllm_moe import formats as fmt

FORMATS = ("mxfp4", "mxfp6")


def _blocks():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, 96, generator=g) * torch.exp2(torch.randint(-30, 30, (64, 1), generator=g).float())
    x[0] = 0
    x[1, :32] = torch.linspace(-8, 8, 32)
    for i, top in enumerate((6.0, 6.999, 7.0, 7.49, 7.5, 7.7499, 7.75, 7.76, 8.0)):   # around what still fits
        x[2 + i] = top * torch.linspace(0, 1, 96)
    x[20] *= 1e-38
    x[21] = 3e38 * torch.linspace(-1, 1, 96)
    x[22] = torch.arange(96) / 16           # ties of both formats
    return x


@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_matches_grid_search(f, dt):
    x = _blocks()
    if dt == torch.float16:
        x = x.clamp(-60000, 60000)
    x = x.to(dt)
    codes, scales = fmt.mx_quantize(x, f)
    b = x.double().reshape(64, 3, 32)
    s = mx_ref.scale_byte(b.abs().amax(-1, keepdim=True), f)
    assert torch.equal(scales.double(), s.squeeze(-1))
    top = 1 << (mx_ref.BITS[f] - 1)
    c = mx_ref.unpack(codes, f)
    assert torch.equal(c & (top - 1), mx_ref.codes_of(b, s, f).reshape(64, 96))
    assert torch.equal((c & top) != 0, torch.signbit(x))
    v = mx_ref.dequant(codes, scales, f)
    assert torch.equal(fmt.mx_dequant(codes, scales, f), v.float())   # fp32: 3e38 becomes 2^128 in mxfp4, an infinity
    # no element is off by more than half a step: 2^-M-1 of it, or of the scale below 1
    half = 2.0 ** -(mx_ref.MANTISSA[f] + 1)
    err = (v.reshape(b.shape) - b).abs()
    assert bool((err <= half * torch.maximum(b.abs(), 2.0 ** (s - 127))).all())


@pytest.mark.parametrize("f", FORMATS)
def test_not_finite_blocks(f):
    x = torch.ones(4, 64)
    x[0, 3], x[1, 40], x[2, 63] = float("nan"), float("inf"), -float("inf")
    codes, scales = fmt.mx_quantize(x, f)
    assert scales[:, 0].tolist() == [255, 125, 125, 125] and scales[:, 1].tolist() == [125, 255, 255, 125]
    v = fmt.mx_dequant(codes, scales, f)
    assert torch.equal(torch.isnan(v), torch.isnan(v.reshape(4, 2, 32)[..., :1]).expand(4, 2, 32).reshape(4, 64))
    assert torch.equal(v[3], x[3]) and bool((codes.reshape(4, 2, -1)[0, 0] == 0).all())


def test_bytes_per_expert():
    assert fmt.bytes_per_expert(3, 2048, 768) == 3 * 2048 * 768 * 17 // 32


# ------------------------------------------------------------------------------------------ refusals
def _rc(name, *args):
    L = nanovllm_moe.capi()
    return getattr(L, name)(*args), L.mi_moe_last_error().decode()


P = ctypes.c_void_p(1 << 12)   # never read: every call below is refused first, or has nothing to do


@pytest.mark.parametrize("args,word", [
    ((P, 3, 4, 64, 64, 0, P, P, None), "fp16, bf16 or fp32"),
    ((P, 1, 4, 64, 64, 2, P, P, None), "format"),
    ((P, 1, 4, 48, 48, 0, P, P, None), "multiple of 32"),
    ((P, 1, 4, 0, 64, 0, P, P, None), "multiple of 32"),
    ((P, 1, -1, 64, 64, 0, P, P, None), "multiple of 32"),
    ((P, 1, 1 << 40, 64, 64, 0, P, P, None), "2^40"),
    ((P, 1, 4, 64, 32, 0, P, P, None), "row_stride"),
    ((P, 1, 4, 64, 68, 0, P, P, None), "row_stride"),
    ((P, 2, 4, 64, 66, 0, P, P, None), "row_stride"),
    ((P, 1, 4, 64, 1 << 41, 0, P, P, None), "row_stride"),
    ((ctypes.c_void_p(4104), 1, 4, 64, 64, 0, P, P, None), "aligned"),
    ((P, 1, 4, 64, 64, 0, ctypes.c_void_p(4104), P, None), "aligned"),
    ((None, 1, 4, 64, 64, 0, P, P, None), "null"),
    ((P, 1, 4, 64, 64, 0, P, None, None), "null"),
])
def test_quantize_refusals(args, word):
    rc, msg = _rc("mi_moe_mx_quantize", *args)
    assert rc == 1 and word in msg, (rc, msg)


@pytest.mark.parametrize("args,word", [
    ((P, P, 4, 64, 0, P, 5, None), "fp16, bf16 or fp32"),
    ((P, P, 4, 64, 7, P, 1, None), "format"),
    ((P, P, 4, 33, 0, P, 1, None), "multiple of 32"),
    ((P, P, 4, 64, 0, ctypes.c_void_p(4104), 1, None), "aligned"),
    ((P, None, 4, 64, 0, P, 1, None), "null"),
])
def test_dequantize_refusals(args, word):
    rc, msg = _rc("mi_moe_mx_dequantize", *args)
    assert rc == 1 and word in msg, (rc, msg)


def test_empty_calls():
    assert _rc("mi_moe_mx_quantize", None, 1, 0, 64, 64, 0, None, None, None)[0] == 0
    assert _rc("mi_moe_mx_dequantize", None, None, 0, 64, 0, None, 1, None)[0] == 0


@pytest.mark.parametrize("E,H,I,word", [(4, 96, 64, "64"), (4, 64, 48, "32"), (4, 1 << 17, 64, "65536"),
                                        (600, 64, 64, "512"), (0, 64, 64, "positive")])
def test_handle_shapes(E, H, I, word):
    h = ctypes.c_void_p()
    rc, msg = _rc("mi_moe_create", E, H, I, 3, ctypes.byref(h))
    assert rc in (1, 3) and word in msg and not h.value, (rc, msg)


def test_no_host_engine():
    h = ctypes.c_void_p()
    mask = (ctypes.c_uint8 * 4)(1, 1, 1, 1)
    rc, msg = _rc("mi_moe_hybrid_create", 4, 64, 64, 3, mask, 1, ctypes.byref(h))
    assert rc == 3 and "MXFP4" in msg
    rc, msg = _rc("mi_moe_cpu_create", 4, 64, 64, 3, 1, 0, ctypes.byref(h))
    assert rc == 3
    nanovllm_moe.load()
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="HIP device"):
            torch.classes.nanovllm.MoEInfer(4, 64, 64, 3)
