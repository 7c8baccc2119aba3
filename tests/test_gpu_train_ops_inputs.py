"""Tensors that are not plain memory of their own, as inputs and outputs of the embedding and clipping operators."""
import pytest
import torch

from codecoder_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_clipping_leaves_the_other_side_of_a_lazy_copy():
    """A copy-on-write tensor shares its memory until one side is written: clipping writes to its own side only."""
    x = torch.randn(5000, device=DEV)
    keep = x.clone()
    y = torch._lazy_clone(x)
    ops.clip_grads([y], 0.5)                                    # in place
    assert torch.equal(x, keep) and abs(float(y.double().norm()) - 0.5) < 1e-5
    y = torch._lazy_clone(x)
    ops.clip_grads([x], 0.5)                                    # in place, on the side that was there first
    assert torch.equal(y, keep) and abs(float(x.double().norm()) - 0.5) < 1e-5
    x.copy_(keep)
    g = torch.randn(5000, device=DEV)
    y = torch._lazy_clone(x)
    ops.clip_grads([g], 0.5, out=[y])                           # as an output
    assert torch.equal(x, keep) and abs(float(y.double().norm()) - 0.5) < 1e-5
    y = torch._lazy_clone(x)
    ops.clip_grads([x], 0.5, out=[y])                           # an output that is a lazy copy of its input
    assert torch.equal(x, keep) and abs(float(y.double().norm()) - 0.5) < 1e-5
    y = torch._lazy_clone(x)
    assert torch.equal(ops.grad_norm([x]), ops.grad_norm([y]))
    assert torch.equal(x, keep) and torch.equal(y, keep)


def test_reading_a_lazy_copy_makes_no_copy():
    w, ids = torch.randn(300, 64, device=DEV), torch.randint(0, 300, (70,), device=DEV)
    gy = torch.randn(70, 64, device=DEV)
    for f in (lambda a, i, g: ops.embed_lookup(i, a), lambda a, i, g: ops.embed_wgrad(g, i, 300),
              lambda a, i, g: ops.grad_norm([a, g])):
        lazy = [torch._lazy_clone(t) for t in (w, ids, gy)]
        want = f(w, ids, gy)
        assert torch.equal(f(*lazy), want)
        assert all(torch._C._is_cow_tensor(t) for t in lazy)
