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


@pytest.mark.parametrize("T", [1, 3001])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_group_with_one_expert_left(dev, score, T):
    """A masked expert is out of its group's sum; the group goes on with those it has left."""
    x = torch.full((T, 64), -INF)
    x[:, 41] = 0.5
    for groups, top in ((8, 1), (8, 3), (16, 2), (16, 1), (4, 3)):
        ids, w = _scores(x.to(dev), 4, None, score, groups, top, 2, True, 1.0)
        assert all(i == [41, -1, -1, -1] for i in ids) and all(v == [1.0, 0.0, 0.0, 0.0] for v in w), (groups, ids[0])
    x[:, 0], x[:, 1], x[:, 41] = -9.0, -9.0, 9.0    # two small choices in one group, a large one alone in another
    ids, _ = _scores(x.to(dev), 2, None, score, 8, 1, 2, False, 1.0)
    assert all(i == [41, -1] for i in ids), ids[0]
    x[:, 0], x[:, 1], x[:, 41] = 1.0, 1.0, 1.1      # two that outweigh one a little larger
    ids, _ = _scores(x.to(dev), 2, None, score, 8, 1, 2, False, 1.0)
    assert all(i == [0, 1] for i in ids), ids[0]


@pytest.mark.parametrize("E,groups,top,K", [(64, 8, 1, 4), (64, 8, 3, 4), (60, 4, 1, 3), (250, 5, 2, 6), (256, 8, 4, 8),
                                            (128, 16, 4, 8), (512, 64, 9, 10), (511, 7, 1, 3)])
@pytest.mark.parametrize("T", [40, 3200])
def test_nothing_routed_to_nothing(dev, E, groups, top, K, T):
    """A token with an expert left is routed to one, and never to a masked one."""
    g = torch.Generator().manual_seed(E + groups)
    x = torch.randn(T, E, generator=g)
    left = torch.randint(1, 5, (T, 1), generator=g)              # experts left in a row
    x[torch.rand(T, E, generator=g).argsort(1).argsort(1) >= left] = -INF
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.randn(E, generator=g), torch.full((E,), -3.0)):
            for group_top in (1, 2):
                ids, _ = torch.ops.nanovllm.moe_topk_scores(x.to(dev), K, None if bias is None else bias.to(dev), score,
                                                            groups, top, group_top, True, 1.0)
                ids = ids.cpu().long()
                n = (ids >= 0).sum(1)
                assert bool((n >= 1).all()), (score, group_top, int((n == 0).sum()))
                assert bool((ids[:, 0] >= 0).all())
                assert bool(torch.gather(x, 1, ids.clamp_min(0))[ids >= 0].isfinite().all())
                groups_left = (x.reshape(T, groups, -1) > -INF).any(-1).sum(1)
                assert bool((n >= torch.minimum(groups_left, torch.tensor(min(top, K)))).all())   # one at least of each group


def test_group_top_without_groups_to_drop(dev):
    """Where every group is taken, group_top has no meaning and no limit but its own: groups of one expert run as they are."""
    f, x = torch.ops.nanovllm.moe_topk_scores, torch.tensor([[0.5, 2.0, -1.0, 1.0]], device=dev)
    ids, w = f(x[:, :1], 1)
    assert ids.tolist() == [[0]] and w.tolist() == [[1.0]]
    for args in ((None, "softmax", 4, 4), (None, "softmax", 4, 4, 1), (None, "softmax")):
        assert f(x, 3, *args)[0].tolist() == [[1, 3, 0]]
    for args in ((None, "softmax", 4, 3), (None, "softmax", 4, 4, 3), (None, "softmax", 4, 4, 0)):
        with pytest.raises(RuntimeError, match="group_top"):
            f(x, 3, *args)
