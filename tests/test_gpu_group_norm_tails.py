"""Group normalisation where the activation's logistic function leaves fp32's normal numbers: z from -200 to 60.  Below u = -87.34
(2^-126) the kernels' s(u) is zero, so z s(u) is off by 2^-126 |z| <= 2^-119 at most, SiLU's |z| being 88 there and GELU's 10, and
the slope s (1 + z u' (1 - s)) by 2^-126 (1 + 88) (GELU: |z u'| <= 3 |u| = 264, 2^-117).  The other terms are test_gpu_group_norm.py's."""
import pytest
import torch

from codecoder_b200 import ops
from test_gpu_group_norm import BF16, EPS, F32, HALF, SUB, definition, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("B,N,C,G", [(300, 1, 64, 8), (40, 50, 64, 8), (2, 9000, 64, 8), (2, 3, 8400, 2)])
def test_biases_far_from_zero(B, N, C, G, act, types):
    x, gy, w, _ = make(B, N, C, *types, True, N + C)
    b = torch.linspace(-200.0, 60.0, C, device=DEV) if act == "silu" else torch.linspace(-25.0, 12.0, C, device=DEV)
    want = definition(x, G, w, b, EPS, act, gy)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.group_norm(*leaves[:1], G, *leaves[1:], EPS, act, types[1])
    grads = torch.autograd.grad(y, leaves, gy)
    xd = x.detach().double().view(B, N, G, C // G)
    rstd = float((xd.var((1, 3), correction=0) + EPS).rsqrt().max())
    top, size = float(gy.double().abs().max()), float(w.detach().abs().max())
    xh = rstd * float(xd.abs().max() + xd.mean((1, 3)).abs().max())
    per = {"y": 2.0**-119, "dx": 2.0**-117 * top * size * rstd * (2 + xh * xh), "dw": 2.0**-117 * B * N * top * xh, "db": 2.0**-117 * B * N * top}
    for what, got, (ref, e), dtype in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), want, (types[1], types[0], F32, F32)):
        e = e + per[what]
        tol = e + (ref.abs() + e) * HALF[dtype] + SUB[dtype]
        err = (got.double() - ref).abs()
        assert bool((err <= tol).all()), (what, float((err / tol).max()))
    assert bool(y.isfinite().all()) and all(bool(g.isfinite().all()) for g in grads)
