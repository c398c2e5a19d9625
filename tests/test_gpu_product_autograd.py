"""The differentiable product as torch's own tools see it: dispatch modes, checkpointing, hooks on saved tensors, and what it
refuses."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import products_ref as ref

pytestmark = pytest.mark.gpu


class _Calls(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "nanovllm":
            self.names.append(func.__name__.split(".")[0])
        return func(*args, **(kwargs or {}))


def _inputs(cuda):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randn(*s, generator=g, device=cuda).to(torch.bfloat16) for s in ((30, 48), (3, 40, 48), (30, 40)))
    return x.requires_grad_(), w.requires_grad_(), dy, torch.tensor([0, 10, 10, 28], dtype=torch.int32, device=cuda)


def _wanted(x, w, dy, s):
    x, w, st = x.detach(), w.detach(), s.tolist()
    return ref.grouped_dx(dy, w, st, x.dtype), ref.grouped_dw(dy, x, st, w.shape[0], x.dtype)


def test_dispatch_modes_see_every_product(cuda):
    x, w, dy, s = _inputs(cuda)
    ops = torch.ops.nanovllm
    for leaves, names in (((x, w), ["moe_grouped_matmul", "moe_grouped_matmul_dx", "moe_grouped_matmul_dw"]),
                          ((x,), ["moe_grouped_matmul", "moe_grouped_matmul_dx"]), ((w,), ["moe_grouped_matmul", "moe_grouped_matmul_dw"])):
        a, b = (t if any(t is l for l in leaves) else t.detach() for t in (x, w))
        with _Calls() as calls:
            grads = torch.autograd.grad(ops.moe_grouped_matmul(a, b, s), leaves, dy)
        assert calls.names == names
        want = {id(x): _wanted(x, w, dy, s)[0], id(w): _wanted(x, w, dy, s)[1]}
        for l, g in zip(leaves, grads):
            assert ref.within(g, *want[id(l)]) <= 1.0
    with torch.no_grad(), _Calls() as calls:
        ops.moe_grouped_matmul(x, w, s)
    assert calls.names == ["moe_grouped_matmul"]


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed(cuda, reentrant):
    """Activation checkpointing runs the forward again, and gives the same bits."""
    from torch.utils.checkpoint import checkpoint
    x, w, dy, s = _inputs(cuda)
    ops = torch.ops.nanovllm

    def f(a):
        return torch.nn.functional.silu(ops.moe_grouped_matmul(a, w, s))

    want = torch.autograd.grad(f(x), (x, w), dy)
    with _Calls() as calls:
        f_x = checkpoint(f, x, use_reentrant=reentrant)
        f_x.backward(dy)
    assert calls.names == ["moe_grouped_matmul"] * 2 + ["moe_grouped_matmul_dx", "moe_grouped_matmul_dw"]
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


def test_selective_checkpoint_keeps_the_product(cuda):
    from functools import partial

    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    x, w, dy, s = _inputs(cuda)
    ops = torch.ops.nanovllm

    def f(a):
        return torch.nn.functional.silu(ops.moe_grouped_matmul(a, w, s))

    def keep(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if op is ops.moe_grouped_matmul.default else CheckpointPolicy.PREFER_RECOMPUTE

    want = torch.autograd.grad(f(x), (x, w), dy)
    with _Calls() as calls:
        y = checkpoint(f, x, use_reentrant=False, context_fn=partial(create_selective_checkpoint_contexts, keep))
        got = torch.autograd.grad(y, (x, w), dy)
    assert calls.names == ["moe_grouped_matmul", "moe_grouped_matmul_dx", "moe_grouped_matmul_dw"]   # not run again
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_saved_tensor_hooks(cuda):
    """What is kept for the backward pass goes through the hooks (to the host and back)."""
    x, w, dy, s = _inputs(cuda)
    seen = []

    def pack(t):
        seen.append(tuple(t.shape))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(cuda)):
        y = torch.ops.nanovllm.moe_grouped_matmul(x, w, s)
    got = torch.autograd.grad(y, (x, w), dy)
    assert sorted(seen) == sorted([(30, 48), (3, 40, 48), (4,)])
    for g, want in zip(got, _wanted(x, w, dy, s)):
        assert ref.within(g, *want) <= 1.0


def test_refused_transforms(cuda):
    """Second derivatives, forward mode and function transforms raise; starts changed before the backward pass too."""
    x, w, dy, s = _inputs(cuda)
    f = torch.ops.nanovllm.moe_grouped_matmul
    y = f(x, w, s)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: f(a, w.detach(), s).float().sum())(x.detach())
    with pytest.raises(RuntimeError), torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)), w.detach(), s)
    y = f(x, w, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(y, x, dy)
