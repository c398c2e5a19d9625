"""Corners of the score router on host and device, against results worked out by hand."""
import math

import pytest
import torch

import nanovllm_moe

INF = float("inf")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def dev(request):
    if request.param == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")
    nanovllm_moe.load()
    return torch.device(request.param)


def _scores(x, *args):
    ids, w = torch.ops.nanovllm.moe_topk_scores(x, *args)
    return ids.tolist(), w.double().tolist()


def _near(got, want):
    """One rounding to fp32 each, and 2^-36 for sums and scores (subnormal ones of some 10^12 steps)."""
    return all(abs(g - w) <= abs(w) * (2.0 ** -24 + 2.0 ** -36) for g, w in zip(got, want))


@pytest.mark.parametrize("T", [1, 3001])
def test_sigmoid_of_very_low_logits(dev, T):
    """Scores far below fp32's range are still scores: sigmoid(l) = exp(l) there, and the picks' ratio is exp(l1 - l2)."""
    x = torch.full((T, 64), -740.0)
    x[:, 5], x[:, 6] = -715.0, -720.0
    ids, w = _scores(x.to(dev), 2, None, "sigmoid", 1, 1, 1, True, 1.0)
    a = 1 / (1 + math.exp(-5.0))
    assert all(i == [5, 6] for i in ids) and all(_near(v, [a, 1 - a]) for v in w), (ids[0], w[0])
    x[:, 6] = -760.0         # below 64 bits' range: a score of 0, as the lower ids' -750
    x[:, :5] = x[:, 7:] = -750.0
    ids, w = _scores(x.to(dev), 3, None, "sigmoid", 1, 1, 1, True, 2.5)
    assert all(i == [5, 0, 1] for i in ids) and all(v == [2.5, 0.0, 0.0] for v in w), (ids[0], w[0])
