"""Expert outputs of MXFP4 layers: rows of the down projection that are far larger than their neighbours leave the
other columns at their own precision, in calls of every size; and weights whose scale bytes the quantizer never writes."""
import pytest
import torch

import mx_layer_ref
import mx_ref
from helpers import topk_routing
from nanovllm_moe import formats as fmt

pytestmark = pytest.mark.gpu

TOKENS = [1, 8, 70, 300]   # decode calls, items of 64 rows, items of 128


def _weights(E, H, I, rows, seed):
    """gate||up and down as codes and scales; down's row n is rows[n] times the others' size."""
    g = torch.Generator().manual_seed(seed)
    w13 = torch.randn(E, 2 * I, H, generator=g) * 0.05
    w2 = torch.randn(E, H, I, generator=g) * 0.05 * rows.reshape(1, H, 1)
    return fmt.mx_quantize(w13, "mxfp4"), fmt.mx_quantize(w2, "mxfp4")


def _handle(E, H, I, a, b, cuda):
    h = torch.classes.nanovllm.MoEInfer(E, H, I, 3)
    h.store_mxfp4_repack(*[t.to(cuda) for t in (*a, *b)])
    return h


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("factor", [30.0, 1000.0, 1e5])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_columns_of_unequal_size(cuda, T, factor, dt):
    E, H, I, K = 8, 192, 96, 4
    rows = torch.ones(H)
    rows[[5, 16, 47, 64, 130, 191]] = factor
    rows[[6, 100]] = 1 / factor
    a, b = _weights(E, H, I, rows / factor ** 0.5, seed=T)
    h = _handle(E, H, I, a, b, cuda)
    ids, tw = topk_routing(T, E, K, seed=T)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dt)
    y = torch.ops.nanovllm.moe_forward(x.to(cuda), ids.to(cuda), tw.to(cuda), h).cpu()
    ref, bound = mx_layer_ref.layer(x.double(), ids, tw.double(), mx_ref.dequant(*a, "mxfp4"), mx_ref.dequant(*b, "mxfp4"), dt)
    r = mx_ref.within(y, ref, bound)
    assert r <= 1.0, r


@pytest.mark.parametrize("T", TOKENS)
def test_one_column_beyond_fp32(cuda, T):
    """Outputs beyond the fp32 range in one column: every other column as without them."""
    E, H, I, K = 4, 192, 96, 2
    a, b = _weights(E, H, I, torch.ones(H), seed=3)
    small, big = b[1].clone(), b[1].clone()
    small[:, 37], big[:, 37] = 0, 254
    ids, tw = topk_routing(T, E, K, seed=T)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16) * 8
    y = [torch.ops.nanovllm.moe_forward(x.to(cuda), ids.to(cuda), tw.to(cuda), _handle(E, H, I, a, (b[0], s), cuda)).cpu()
         for s in (small, big)]
    keep = torch.arange(H) != 37
    assert torch.equal(y[0][:, keep], y[1][:, keep]) and bool(y[0].isfinite().all())
    assert not bool(y[1][:, 37].isfinite().any())


@pytest.mark.parametrize("E,H,I,K", [(4, 64, 32, 3), (5, 512, 256, 2), (16, 320, 416, 4), (64, 256, 128, 10), (64, 192, 96, 16)])
@pytest.mark.parametrize("T", [1, 3, 6, 17, 65, 200])
def test_layer_in_fp32(cuda, E, H, I, K, T):
    """Calls of every path within the bound of fp32 sums and outputs, held to each element."""
    a, b = _weights(E, H, I, torch.ones(H), seed=E + I)
    h = _handle(E, H, I, a, b, cuda)
    ids, tw = topk_routing(T, E, K, seed=T)
    dt = torch.bfloat16 if T % 2 else torch.float16
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dt)
    y = torch.ops.nanovllm.moe_forward(x.to(cuda), ids.to(cuda), tw.to(cuda), h).cpu()
    ref, bound = mx_layer_ref.layer(x.double(), ids, tw.double(), mx_ref.dequant(*a, "mxfp4"), mx_ref.dequant(*b, "mxfp4"), dt)
    r = mx_ref.within(y, ref, bound)
    assert r <= 1.0, r


# ------------------------------------------------------------------------------------------ scale bytes
@pytest.mark.parametrize("T", TOKENS)
def test_scale_bytes_of_any_size(cuda, T):
    """Scales that differ widely from block to block, and 0 and 254 among them: the layer of the values they stand for."""
    E, H, I, K = 4, 192, 96, 2
    g = torch.Generator().manual_seed(T)
    codes = [torch.randint(0, 256, s, generator=g, dtype=torch.uint8) for s in ((E, 2 * I, H // 2), (E, H, I // 2))]
    s13 = torch.randint(112, 124, (E, 2 * I, H // 32), generator=g)
    s2 = torch.randint(87, 168, (E, H, I // 32), generator=g)
    s13[:, ::7, 1], s2[:, ::5, 2] = 0, 0                    # 2^-127: nothing beside the others
    s13[:, 1::9, 3], s2[:, 2::11, 0] = 254, 254             # 2^127 of zeros: nothing at all
    codes[0].view(E, 2 * I, H // 32, 16)[:, 1::9, 3] = 0
    codes[1].view(E, H, I // 32, 16)[:, 2::11, 0] = 0
    a, b = (codes[0], s13.to(torch.uint8)), (codes[1], s2.to(torch.uint8))
    h = _handle(E, H, I, a, b, cuda)
    ids, tw = topk_routing(T, E, K, seed=T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    y = torch.ops.nanovllm.moe_forward(x.to(cuda), ids.to(cuda), tw.to(cuda), h).cpu()
    ref, bound = mx_layer_ref.layer(x.double(), ids, tw.double(), mx_ref.dequant(*a, "mxfp4"), mx_ref.dequant(*b, "mxfp4"), x.dtype)
    r = mx_ref.within(y, ref, bound)
    assert r <= 1.0, r


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T", TOKENS)
def test_scale_byte_255(cuda, T, zeros):
    """A block of scale 255 makes its products NaN, whatever its codes: in gate or up the tokens of that expert, in down
    one column of theirs, and nothing else."""
    E, H, I, K = 6, 192, 96, 2
    a, b = _weights(E, H, I, torch.ones(H), seed=9)
    clean = _handle(E, H, I, a, b, cuda)
    a, b = [t.clone() for t in a], [t.clone() for t in b]
    for p, e, row, block in ((a, 0, 5, 5), (a, 1, I + 95, 0), (b, 2, 7, 1), (b, 3, 191, 2)):
        p[1][e, row, block] = 255
        if zeros:
            p[0][e, row, 16 * block:16 * block + 16] = 0
    h = _handle(E, H, I, a, b, cuda)
    ids, tw = topk_routing(T, E, K, seed=T)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(cuda)
    y, want = (torch.ops.nanovllm.moe_forward(x, ids.to(cuda), tw.to(cuda), v).cpu() for v in (h, clean))
    nan = (ids < 2).any(1, keepdim=True).expand(T, H).clone()
    nan[:, 7] |= (ids == 2).any(1)
    nan[:, 191] |= (ids == 3).any(1)
    assert torch.equal(y.isnan(), nan)
    assert torch.equal(y[~nan], want[~nan])
