"""Group normalisation's long sums, u = 2^-24.  Wide groups (no activation, fp32): with sums in 64 bits the mean is off by its
rounding, u |mean|; x - mean by u |x - mean| more; the variance by the factor 2 u and its rounding and eps's addition 2 u more,
so 1 / sqrt(var + eps) by half of that and three roundings of the root and the quotient, at most 6 u; xh by those, its own
rounding and the difference's, 8 u |xh| + u |mean| rstd; y by w times that and a rounding.  Backwards a = gy w rounds once, the
means of a and a xh are off by the means of their terms' errors and a rounding, and dx = rstd (a - (s1 + xh s2)) rounds each of
its operations once."""
import pytest
import torch

from codecoder_b200 import ops
from test_gpu_group_norm import EPS, F32, U, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("shape", [(1, 20000, 1021, 1), (2, 5000, 2052, 1), (1, 7000, 1034, 2)])
@pytest.mark.parametrize("offset", [0.5, 30.0])
def test_wide_groups_of_many_rows(shape, offset):
    B, N, C, G = shape
    x, gy, w, b = make(B, N, C, F32, F32, True, N)
    x += offset                                         # a mean that is not zero grows the partial sums
    gy += 0.1
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.group_norm(x, G, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, leaves, gy)
    xd, gd = (t.detach().double().view(B, N, G, C // G) for t in (x, gy))
    wd, bd = (t.detach().double().view(G, C // G) for t in (w, b))
    mean = xd.mean((1, 3), keepdim=True)
    rstd = ((xd - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    xh = (xd - mean) * rstd
    e_xh = 8 * U * xh.abs() + U * mean.abs() * rstd
    want = xh * wd + bd
    err = (y.detach().double().view_as(want) - want).abs()
    tol = wd.abs() * e_xh + U * want.abs() + U * (wd * xh).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    del err, tol, want
    a = gd * wd
    s1, s2 = a.mean((1, 3), keepdim=True), (a * xh).mean((1, 3), keepdim=True)
    e_s1 = 2 * U * a.abs().mean((1, 3), keepdim=True)
    e_s2 = (a.abs() * e_xh + 2 * U * (a * xh).abs()).mean((1, 3), keepdim=True)
    want = rstd * (a - s1 - xh * s2)
    tol = rstd * (2 * U * a.abs() + e_s1 + 2 * U * s1.abs() + xh.abs() * e_s2 + e_xh * s2.abs() + 2 * U * (xh * s2).abs()) + 8 * U * want.abs()
    err = (dx.double().view_as(want) - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # dw and db: sums in 64 bits of values that are off as above
    e_dw = (gd.abs() * e_xh).sum((0, 1)) + U * (gd * xh).abs().sum((0, 1))
    assert bool(((dw.double().view(G, -1) - (gd * xh).sum((0, 1))).abs() <= e_dw).all())
    assert bool(((db.double().view(G, -1) - gd.sum((0, 1))).abs() <= U * gd.abs().sum((0, 1))).all())


@pytest.mark.parametrize("B,C,G", [(60_000, 16_384, 32), (60_000, 8192, 4), (150_000_000, 4, 1)])
def test_a_bias_gradient_over_many_samples(B, C, G):
    """Gradients that are all alike, whose roundings do not cancel: a thread adds up 256 samples at most, 256 u, and what the
    threads have joins in 64 bits, rounded to fp32 twice."""
    x = torch.zeros(B, 1, C, device=DEV)
    x[:, :, ::2] = 1.0
    b = torch.zeros(C, device=DEV, requires_grad=True)
    gy = torch.full((B, 1, C), 0.1, device=DEV)
    db, = torch.autograd.grad(ops.group_norm(x, G, None, b), b, gy)
    want = B * float(gy[0, 0, 0].double())
    assert float((db.double() - want).abs().max()) <= 258 * U * want
