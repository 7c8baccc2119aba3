"""RoundMemory on a padded batch: what stands behind a shot's rounds, whatever it is, reaches no result but its own."""
import pytest
import torch

from test_gpu_layers import make_memory

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("T", [9, 70])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1e30])
def test_what_stands_behind_a_shots_rounds_reaches_no_gradient(T, value, autocast):
    B, S, C = 4, 5, 64
    m = make_memory(C, 2, S, T)
    n = torch.tensor([T, 0, T // 2, 1], device=DEV)
    dead = torch.arange(T, device=DEV) >= n[:, None]
    x, gy = torch.randn(2, B, T, S, C, device=DEV)
    out = []
    for fill in (0.0, value):
        xs = torch.where(dead[:, :, None, None], torch.full_like(x, fill), x).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y, state = m(xs, lengths=n, return_state=True)
        live = torch.where(dead[:, :, None, None], 0, y)
        assert torch.equal(y[dead].isnan(), xs[dead].isnan()) and torch.equal(y[dead].nan_to_num(), xs[dead].nan_to_num())
        grads = torch.autograd.grad(y, [xs, *m.parameters()], gy.to(y.dtype))
        assert torch.equal(grads[0][dead], gy.to(y.dtype)[dead].to(x.dtype))         # passed through
        out.append((live, state, *grads))
    for a, b in zip(*out):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
