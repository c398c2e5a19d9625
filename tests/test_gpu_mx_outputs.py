"""Expert outputs of MXFP4 layers: rows of the down projection that are far larger than their neighbours leave the
other columns at their own precision, in calls of every size."""
import pytest
import torch

import mx_layer_ref
import mx_ref
import nanovllm_moe
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
