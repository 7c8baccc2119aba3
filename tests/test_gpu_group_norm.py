"""Group normalisation with an activation on the GPU, and its gradients, against the definition in 64 bits.

Tolerances, u = 2^-24.  A statistic over M values adds them in chains of at most D = ceil(M / 128) + 32 roundings, so the mean
is off by e_mu <= (D + 2) u mean|x| + u |mean|, the variance (squared differences) by (D + 4) u var + e_mu^2, hence
rstd by the factor e_r = half of that over (var + eps), + 3 u, and xh by e_xh = rstd e_mu + |xh| (e_r + 3 u).  z adds two
roundings.  The logistic function of an argument a takes an exponential of relative error (4 + 2.4 |a|) u and an argument
that is off by 4 u |a| (GELU): s is off by the factor (1 - s) (4 + 7 |a|) u + 6 u.  |act'| <= 1.13 and |act''| <= 1.2.  The
gradients follow by the product rule and the same sums; the sums over rows of dw and db run in chains of at most
rows / 32 + 128 roundings.  Each result is rounded once to its type: half a step relative to the value."""
import math

import pytest
import torch

from codecoder_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0**-24
HALF = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}
SUB = {F32: 2.0**-126, BF16: 2.0**-126, F16: 2.0**-25}
EPS = 1e-5


def make(B, N, C, x_dtype, y_dtype, affine, seed, offset=0.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(B, N, C, generator=g, device=DEV) * 1.5 + offset * torch.randn(C, generator=g, device=DEV)).to(x_dtype)
    gy = (torch.randn(B, N, C, generator=g, device=DEV) / 8).to(y_dtype)
    w = 1 + 0.2 * torch.randn(C, generator=g, device=DEV) if affine else None
    b = 0.3 * torch.randn(C, generator=g, device=DEV) if affine else None
    return x, gy, w, b


def definition(x, G, w, b, eps, act, gy=None):
    """Values and error bounds in 64 bits: (y, e_y) and with gy also dx, dw, db and theirs."""
    B, N, C = x.shape
    M, D = N * C // G, math.ceil(N * C // G / 128) + 32
    xd = x.double().view(B, N, G, C // G)
    mean = xd.mean((1, 3), keepdim=True)
    xc = xd - mean
    var = (xc * xc).mean((1, 3), keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = xc * rstd
    e_mu = (D + 2) * U * xd.abs().mean((1, 3), keepdim=True) + U * mean.abs()
    e_r = 0.5 * ((D + 4) * U * var + e_mu**2) / (var + eps) + 3 * U
    e_xh = rstd * e_mu + xh.abs() * (e_r + 3 * U)
    wd = torch.ones(C, device=x.device, dtype=torch.float64) if w is None else w.double()
    wd = wd.view(G, C // G)
    bd = torch.zeros_like(wd) if b is None else b.double().view(G, C // G)
    z = xh * wd + bd
    e_z = wd.abs() * e_xh + 2 * U * ((xh * wd).abs() + z.abs())
    if act == "none":
        a, da, s = z, torch.ones_like(z), torch.ones_like(z)
    else:
        a = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)
        da = torch.ones_like(z) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z**2)
        s = torch.sigmoid(a)
    y = z * s
    c = 0 if act == "none" else (1 - s) * (4 + 7 * a.abs()) * U + 6 * U
    e_y = 1.13 * e_z + y.abs() * c
    out = [(y.view(B, N, C), e_y.view(B, N, C))]
    if gy is None:
        return out
    slope = torch.ones_like(z) if act == "none" else s + z * s * (1 - s) * da
    gyd = gy.double().view(B, N, G, C // G)
    gz = gyd * slope
    e_gz = gyd.abs() * (1.2 * e_z + (s + (z * s * (1 - s) * da).abs()) * (c + 8 * U)) + U * gz.abs()
    av, e_a = gz * wd, e_gz * wd.abs() + U * (gz * wd).abs()
    s1, s2 = av.mean((1, 3), keepdim=True), (av * xh).mean((1, 3), keepdim=True)
    e_s1 = e_a.mean((1, 3), keepdim=True) + (D + 4) * U * av.abs().mean((1, 3), keepdim=True)
    e_s2 = (e_a * xh.abs() + av.abs() * e_xh).mean((1, 3), keepdim=True) + (D + 5) * U * (av * xh).abs().mean((1, 3), keepdim=True)
    dx = rstd * (av - s1 - xh * s2)
    e_dx = rstd * (e_a + e_s1 + xh.abs() * e_s2 + e_xh * s2.abs() + 4 * U * (av.abs() + s1.abs() + (xh * s2).abs())) \
        + dx.abs() * (e_r + 2 * U)
    out.append((dx.view(B, N, C), e_dx.view(B, N, C)))
    R = math.ceil(B * N / 32) + 128
    dw = (gz * xh).sum((0, 1)).view(C)
    e_dw = ((e_gz * xh.abs() + gz.abs() * e_xh).sum((0, 1)) + R * U * (gz * xh).abs().sum((0, 1))).view(C)
    db = gz.sum((0, 1)).view(C)
    e_db = (e_gz.sum((0, 1)) + R * U * gz.abs().sum((0, 1))).view(C)
    return out + [(dw, e_dw), (db, e_db)]


def check(got, want, dtype, what):
    ref, e = want
    assert got.dtype == dtype and got.shape == ref.shape, what
    tol = e + (ref.abs() + e) * HALF[dtype] + SUB[dtype]
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def run(B, N, C, G, act, x_dtype, y_dtype, affine, seed, offset=0.5, views=None):
    x, gy, w, b = make(B, N, C, x_dtype, y_dtype, affine, seed, offset)
    if views is not None:
        x, gy = views(x), views(gy)
    want = definition(x, G, w, b, EPS, act, gy)
    with torch.no_grad():
        check(ops.group_norm(x, G, w, b, EPS, act, y_dtype), want[0], y_dtype, "y")
    leaves = [x.detach()] + ([w, b] if affine else [])
    leaves = [t.requires_grad_() for t in leaves]
    y = ops.group_norm(leaves[0], G, *(leaves[1:] if affine else (None, None)), EPS, act, y_dtype)
    check(y.detach(), want[0], y_dtype, "y with gradients")
    grads = torch.autograd.grad(y, leaves, gy)
    check(grads[0], want[1], x_dtype, "dx")
    if affine:
        check(grads[1], want[2], F32, "dw")
        check(grads[2], want[3], F32, "db")


SHAPES = [(1, 1, 4, 1), (1, 1, 512, 32), (3, 1, 96, 3), (777, 1, 96, 3), (5, 1, 1000, 8), (4100, 1, 24, 3), (257, 1, 160, 5),
          (2, 2, 64, 8), (300, 7, 32, 4), (1, 504, 512, 32), (37, 333, 45, 5), (3, 504, 128, 8), (2, 2197, 128, 1),
          (6, 121, 96, 32), (1, 30000, 8, 2), (2, 1500, 1024, 4), (150, 50, 72, 9), (1, 3, 1021, 1), (2, 4097, 6, 3),
          (9, 300, 256, 256), (1, 9000, 516, 1)]
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (F32, F16)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_values_and_gradients_match_the_definition(shape, act):
    k = SHAPES.index(shape) + len(act)
    run(*shape, act, *TYPES[k % 5], affine=k % 4 != 0, seed=k)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(40, 33, 64, 4), (1000, 1, 64, 4), (2, 40000, 64, 2)])
def test_every_type(types, shape):
    run(*shape, "silu", *types, affine=True, seed=11)


def test_a_large_mean_keeps_the_variance():
    run(4, 100, 64, 4, "none", F32, F32, True, 3, offset=1000.0)
    run(400, 1, 64, 2, "silu", F32, F32, True, 4, offset=300.0)


@pytest.mark.parametrize("N", [1, 60])
def test_layouts(N):
    def rows_of_wider(t):
        wide = torch.full((t.shape[0], N + 3, t.shape[2] + 5), 1e9, device=DEV, dtype=t.dtype)
        wide[:, 1:N + 1, 2:-3] = t
        return wide[:, 1:N + 1, 2:-3]
    views = [rows_of_wider, lambda t: t.transpose(0, 2).contiguous().transpose(0, 2), lambda t: t[:1].expand_as(t),
             lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)]
    for i, v in enumerate(views):
        for types in ((F32, BF16), (BF16, BF16)):
            run(6, N, 72, 3, "silu", *types, True, 20 + i, views=v)
    x = torch.randn(4, 3, 5, 32, device=DEV)
    assert torch.equal(ops.group_norm(x, 4), ops.group_norm(x.view(4, 15, 32), 4).view(x.shape))
    assert torch.equal(ops.group_norm(x.view(60, 32), 4), ops.group_norm(x.view(60, 1, 32), 4).view(60, 32))
    y = ops.group_norm(x[:, :, ::2], 4)                            # samples whose positions are no single run
    assert torch.equal(y, ops.group_norm(x[:, :, ::2].contiguous(), 4))


@pytest.mark.parametrize("N,C,G", [(1, 96, 3), (40, 64, 4), (700, 16, 1)])
def test_offsets_past_32_bits(N, C, G):
    """Samples more than 2^31 elements apart (rows and gradients too)."""
    def far(t):
        wide = torch.empty(2**31 + 2**20 + N * C, device=DEV, dtype=t.dtype)
        v = wide.as_strided(t.shape, (2**31 + 2**20, C, 1))
        return v.copy_(t)
    run(2, N, C, G, "silu", BF16, BF16, True, N, views=far)


def test_a_bias_without_a_weight():
    x, gy, w, b = make(9, 31, 24, F32, F32, True, 2)
    x, b = x.requires_grad_(), b.requires_grad_()
    dx, db = torch.autograd.grad(ops.group_norm(x, 3, None, b, EPS, "gelu"), (x, b), gy)
    one = torch.ones(24, device=DEV)
    want = definition(x.detach(), 3, one, b.detach(), EPS, "gelu", gy)
    check(dx, want[1], F32, "dx")
    check(db, want[3], F32, "db")


def test_many_samples_and_many_groups():
    run(70000, 2, 16, 2, "silu", BF16, BF16, True, 1)          # more samples than a grid has rows of blocks
    run(66000, 40, 6, 2, "none", F32, F32, True, 2)
    run(1, 3, 8192, 4096, "silu", F32, BF16, True, 3)
    run(2, 1, 100000, 100000, "none", F32, F32, True, 4)
    run(1, 5, 9000, 3, "gelu", BF16, BF16, True, 5)            # groups wider than a row of threads


def test_empty_tensors():
    w = torch.ones(8, device=DEV, requires_grad=True)
    for shape in ((0, 5, 8), (3, 0, 8), (0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = ops.group_norm(x, 2, w, w.detach())
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert y.shape == shape and dx.shape == shape and bool((dw == 0).all())


@pytest.mark.parametrize("N,C,G", [(1, 64, 4), (50, 64, 4), (20000, 16, 4)])
def test_special_values_stay_in_their_group(N, C, G):
    x = torch.randn(3, N, C, device=DEV)
    ref = ops.group_norm(x, G, activation="silu")
    bad = x.clone()
    bad[1, N // 2, C // G] = float("inf")
    bad[2, 0, 0] = float("nan")
    y = ops.group_norm(bad, G, activation="silu")
    touched = torch.zeros(3, 1, C, dtype=torch.bool, device=DEV)
    touched[1, :, C // G:2 * C // G] = True
    touched[2, :, :C // G] = True
    assert torch.equal(y[~touched.expand_as(y)], ref[~touched.expand_as(y)])
    assert bool(y[2, :, :C // G].isnan().all()) and bool(y[1, N // 2, C // G].isnan())
    const = torch.full((2, N, C), 3.0, device=DEV)
    assert bool((ops.group_norm(const, G) == 0).all())              # no variance: eps keeps it finite


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,G", [(1, 64, 4), (1, 45, 5), (50, 64, 4), (2000, 64, 4), (20000, 16, 4), (2, 4096, 2)])
def test_gradients_of_special_values_stay_in_their_group(N, C, G, dtype):
    """NaN (of the bits that arithmetic makes, and of others) and infinities in x or gy: not finite in all of their group's dx
    and their channels' dw, and elsewhere as they were."""
    x, gy, w, b = make(5, N, C, dtype, dtype, True, N + C)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    clean = torch.autograd.grad(ops.group_norm(x, G, w, b, EPS, "silu"), leaves, gy)
    zero = torch.zeros((), device=DEV)
    made = (zero / zero).to(dtype)                      # 0x7fffffff
    cg = C // G
    bad, bad_g = x.detach().clone(), gy.clone()
    bad[1, N // 2, cg] = float("inf")
    bad[2, 0, 0] = made
    bad_g[3, N - 1, C - 1] = made
    bad_g[4, 0, C - 1] = -float("inf")
    bad.requires_grad_()
    got = torch.autograd.grad(ops.group_norm(bad, G, w, b, EPS, "silu"), [bad, w, b], bad_g)
    touched = torch.zeros(5, 1, C, dtype=torch.bool, device=DEV)
    touched[1, :, cg:2 * cg] = touched[2, :, :cg] = touched[3:, :, C - cg:] = True
    rest = ~touched.expand_as(x)
    assert torch.equal(got[0][rest], clean[0][rest])
    assert not bool(got[0][2, :, :cg].isfinite().any()) and not bool(got[0][3:, :, C - cg:].isfinite().any())
    channels = ~touched.any(0)[0]
    for a_, b_ in zip(got[1:], clean[1:]):
        assert torch.equal(a_[channels], b_[channels])
        assert not bool(a_[C - 1].isfinite())
    assert not bool(got[1][:cg].isfinite().any())


def test_gradients_match_differences():
    torch.manual_seed(5)
    for N, C, G, act in ((1, 12, 2, "silu"), (9, 10, 5, "gelu"), (700, 4, 2, "silu")):
        x, w, b, gy, dx_, dw_, db_ = (torch.randn(s, device=DEV, dtype=torch.float64) for s in
                                      ((2, N, C), C, C, (2, N, C), (2, N, C), C, C))
        gy32 = gy.float()

        def loss(x, w, b):
            y = definition(x, G, w, b, EPS, act)[0][0]
            return float((y * gy32.double()).sum())
        h = 1e-5
        diff = (loss(x + h * dx_, w + h * dw_, b + h * db_) - loss(x - h * dx_, w - h * dw_, b - h * db_)) / (2 * h)
        leaves = [t.float().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(ops.group_norm(leaves[0], G, *leaves[1:], EPS, act), leaves, gy32)
        got = sum(float((g.double() * d).sum()) for g, d in zip(grads, (dx_, dw_, db_)))
        size = sum(float((g.double() * d).abs().sum()) for g, d in zip(grads, (dx_, dw_, db_)))
        # the gradients' errors (about 100 u of their terms) and the inputs' rounding to fp32 (u of every element)
        assert abs(got - diff) <= 1e-5 * size + 1e-5, (got, diff, size)


@pytest.mark.parametrize("shape", [(500, 1, 96, 3), (30, 200, 64, 8), (2, 9000, 64, 2)])
def test_repeats_bit_for_bit_on_any_stream_and_from_graphs(shape):
    B, N, C, G = shape
    x, gy, w, b = make(B, N, C, BF16, BF16, True, 1)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = ops.group_norm(x, G, w, b, EPS, "silu")
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
        once()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once()
        graphs.append((g, out))
    with torch.no_grad():
        x.mul_(0.5), gy.mul_(2.0)
    second = once()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, second))


def test_only_the_gradients_asked_for():
    x, gy, w, b = make(20, 30, 48, F32, F32, True, 7)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.group_norm(full[0], 4, *full[1:], EPS, "silu"), full, gy)
    for k in range(3):
        t = [x, w, b]
        t[k] = t[k].clone().requires_grad_()
        got, = torch.autograd.grad(ops.group_norm(t[0], 4, t[1], t[2], EPS, "silu"), t[k], gy)
        assert torch.equal(got, want[k])
    w16 = w.bfloat16().requires_grad_()
    dw, = torch.autograd.grad(ops.group_norm(x, 4, w16, None), w16, gy)
    assert dw.dtype == BF16


def test_refusals():
    x = torch.randn(4, 5, 12, device=DEV)
    with pytest.raises(ValueError, match="divide"):
        ops.group_norm(x, 5)
    with pytest.raises(ValueError, match="divide"):
        ops.group_norm(x, 0)
    with pytest.raises(ValueError, match="activation"):
        ops.group_norm(x, 3, activation="relu")
    with pytest.raises(ValueError, match="channels"):
        ops.group_norm(x, 3, torch.ones(11, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm(x, 3, torch.ones(12))
    with pytest.raises(TypeError, match="narrows"):
        ops.group_norm(x.half(), 3, dtype=F32)
    with pytest.raises(TypeError, match="group_norm takes"):
        ops.group_norm(x.double(), 3)
    with pytest.raises(RuntimeError, match="eps"):
        ops.group_norm(x, 3, eps=-1.0)
    with pytest.raises(ValueError, match="samples"):
        ops.group_norm(x[0, 0], 3)
    x.requires_grad_()
    g, = torch.autograd.grad(ops.group_norm(x, 3).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
