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


def test_lazily_negated_views():
    """The imaginary part of a conjugate is a view whose values are the negative of its memory."""
    z = torch.randn(40, 1, device=DEV, dtype=torch.complex64).conj()
    w = z.imag                                                  # one channel: no layout asks for a copy
    ids = torch.randint(0, 40, (200,), device=DEV)
    assert w.is_neg() and torch.equal(ops.embed_lookup(ids, w), w.resolve_neg()[ids])
    gy = torch._neg_view(torch.randint(-3, 4, (200, 8), device=DEV).float())
    for V in (5, 40):
        want = torch.zeros(V, 8, device=DEV).index_add_(0, ids % V, gy.resolve_neg())
        assert torch.equal(ops.embed_wgrad(gy, ids % V, V), want)
    x = torch.randn(300, device=DEV)
    keep, neg = x.clone(), torch._neg_view(x)
    n = ops.grad_norm([neg])
    assert torch.equal(n, ops.grad_norm([x]))
    with pytest.raises(ValueError, match="negated"):
        ops.clip_grads([neg], 0.5, out=[torch.empty_like(x)])
    with pytest.raises(ValueError, match="negated"):
        ops.clip_grads([keep], 0.5, out=[neg])
    assert torch.equal(x, keep)
    assert torch.equal(ops.clip_grads([neg], 0.5), n)           # in place: both sides of the view are scaled
    coef = 0.5 / float(n)
    assert float((neg - -keep * coef).abs().max()) < 1e-6 and float((x - keep * coef).abs().max()) < 1e-6
