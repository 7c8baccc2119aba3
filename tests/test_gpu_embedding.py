"""The embedding lookup and its weight gradient on the GPU against their definitions in 64 bits.

Tolerances.  lookup: the fp32 product is off by at most half a step of fp32 (2^-24 relative) and the result by half a
step of its type, plus half of the type's smallest subnormal.  gradient: a sum of m rows in fp32 (any order, partial sums
included, at most m + 1 additions of which each rounds once) is off by at most (m + 1) 2^-24 sum |x|; the scale's product
2^-24 and the type's rounding relative to the value; plus half of the type's smallest subnormal."""
import pytest
import torch

from codecoder_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}
SUB = {F32: 2.0**-150, BF16: 2.0**-134, F16: 2.0**-25}        # half the smallest subnormal


def make_ids(n, V, kind, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        t = torch.randint(0, V, (n,), generator=g)
    elif kind == "padded":                                    # outside on both sides, far ones among them
        t = torch.randint(-2, V + 2, (n,), generator=g)
        far = 2**31 - 1 if dtype == torch.int32 else 2**40 + 1
        t[::7] = far
        t[3::11] = -far
    elif kind == "one":
        t = torch.full((n,), V // 2)
    elif kind == "last":
        t = torch.full((n,), V - 1)
    elif kind == "none":
        t = torch.full((n,), -1)
    elif kind == "hot":                                       # half the rows on one token
        t = torch.randint(0, V, (n,), generator=g)
        t[torch.rand(n, generator=g) < 0.5] = V // 3
    else:                                                     # descending runs
        t = (torch.arange(n).flip(0) * V) // max(n, 1)
    return t.to(dtype).to(DEV)


def check_lookup(y, ids, w, scale, dtype):
    V = w.shape[0]
    i = ids.long()
    ok = (i >= 0) & (i < V)
    ref = w.double()[i.clamp(0, V - 1)] * scale * ok[..., None]
    assert y.dtype == dtype and y.shape == (*ids.shape, w.shape[1])
    err = (y.double() - ref).abs()
    assert bool((err <= ref.abs() * (HALF[dtype] * (1 + 2.0**-20) + 2.0**-24) + SUB[dtype]).all()), float(err.max())
    assert bool((y[~ok] == 0).all())


def check_wgrad(dw, gy, ids, V, scale, dtype):
    C = gy.shape[-1]
    x, i = gy.reshape(-1, C).double().cpu(), ids.reshape(-1).long().cpu()
    ok = (i >= 0) & (i < V)
    x, i = x[ok], i[ok]
    ref = torch.zeros(V, C, dtype=torch.float64).index_add_(0, i, x) * scale
    mag = torch.zeros(V, C, dtype=torch.float64).index_add_(0, i, x.abs()) * abs(scale)
    m = torch.bincount(i, minlength=V).double()[:, None]
    assert dw.dtype == dtype and dw.shape == (V, C)
    err = (dw.double().cpu() - ref).abs()
    tol = (m + 1) * 2.0**-24 * mag
    tol = tol + (ref.abs() + tol) * (HALF[dtype] + 2.0**-24) + SUB[dtype]
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-300)).max())
    assert bool((dw.cpu()[m[:, 0] == 0] == 0).all())


@pytest.mark.parametrize("wt,yt", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (5, 3, 7), (504, 5, 512), (1000, 300, 45), (63, 1000, 96), (4097, 50, 100),
                                   (33, 7, 1100)])
def test_lookup_matches_the_definition(n, V, C, wt, yt):
    g = torch.Generator(device=DEV).manual_seed(n + V)
    w = torch.randn(V, C, generator=g, device=DEV).to(wt)
    for kind, it, scale in (("uniform", torch.int64, 1.0), ("padded", torch.int32, 32.0), ("padded", torch.int64, -0.3)):
        ids = make_ids(n, V, kind, n, it)
        check_lookup(ops.embed_lookup(ids, w, scale, yt), ids, w, scale, yt)


def test_lookup_shapes_strides_and_exact_copies():
    w = torch.randn(37, 64, device=DEV)
    ids = torch.randint(0, 37, (3, 4, 5), device=DEV)
    assert torch.equal(ops.embed_lookup(ids, w), torch.nn.functional.embedding(ids, w))      # scale 1: a copy
    assert torch.equal(ops.embed_lookup(ids.transpose(0, 2), w), w[ids.transpose(0, 2)])
    assert torch.equal(ops.embed_lookup(ids[..., ::2], w), w[ids[..., ::2]])
    big = torch.randn(37, 200, device=DEV)
    for view in (big[:, 3:67], big[:, ::3], big.t()[:37, :30], big[5:6].expand(37, 200), big[::2]):
        i = ids % view.shape[0]
        assert torch.equal(ops.embed_lookup(i, view), view[i])
    one = torch.tensor(4, device=DEV)
    assert torch.equal(ops.embed_lookup(one, w), w[4])
    assert ops.embed_lookup(ids[:0], w).shape == (0, 4, 5, 64)
    assert ops.embed_lookup(ids, w[:, :0]).shape == (3, 4, 5, 0)
    special = torch.tensor([[float("inf"), float("nan"), -0.0, 1e-45], [1.0, 2.0, 3.0, 4.0]], device=DEV)
    got = ops.embed_lookup(torch.tensor([0, 1, -1], device=DEV), special)
    assert torch.equal(got[0].nan_to_num(7.0), special[0].nan_to_num(7.0)) and bool(got[0, 1].isnan())
    assert torch.equal(got[1], special[1]) and bool((got[2] == 0).all())


SHAPES = [(1, 1, 1), (1, 5, 512), (2, 1, 8), (31, 300, 3), (32, 2, 96), (33, 5, 45), (504, 5, 512), (1000, 4, 96),
          (4095, 255, 16), (4096, 256, 64), (4097, 257, 100), (9000, 70000, 24), (20000, 17, 260), (12345, 3000, 1100),
          (300, 1, 2048)]


@pytest.mark.parametrize("n,V,C", SHAPES)
@pytest.mark.parametrize("kind", ["uniform", "padded", "one", "last", "none", "hot", "runs"])
def test_wgrad_matches_the_definition(n, V, C, kind):
    k = SHAPES.index((n, V, C)) + len(kind)
    gt, dt = [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16), (F32, BF16), (F32, F16), (F16, F32)][k % 7]
    it = [torch.int64, torch.int32][k % 2]
    scale = [1.0, 0.5, -3.0][k % 3]
    g = torch.Generator(device=DEV).manual_seed(k)
    gy = (torch.randn(n, C, generator=g, device=DEV) / 8).to(gt)
    ids = make_ids(n, V, kind, k, it)
    check_wgrad(ops.embed_wgrad(gy, ids, V, scale, dt), gy, ids, V, scale, dt)


@pytest.mark.parametrize("gt", [F32, BF16, F16])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_wgrad_every_type(gt, dt):
    for n, V, C in ((700, 6, 72), (700, 600, 72), (700, 600, 71)):
        gy = (torch.randn(n, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) / 8).to(gt)
        ids = make_ids(n, V, "padded", 5)
        check_wgrad(ops.embed_wgrad(gy, ids, V, 1.0, dt), gy, ids, V, 1.0, dt)


@pytest.mark.parametrize("n,V,C", [(300000, 4, 96), (300000, 40, 32), (200000, 100000, 64), (70000, 5, 512),
                                   (65536, 1 << 17, 8)])
def test_wgrad_long_sums_are_right_and_repeat_bit_for_bit(n, V, C):
    gy = torch.randn(n, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(BF16)
    for kind in ("uniform", "hot", "one"):
        ids = make_ids(n, V, kind, 3)
        a = ops.embed_wgrad(gy, ids, V)
        check_wgrad(a, gy, ids, V, 1.0, F32)
        assert torch.equal(a, ops.embed_wgrad(gy, ids, V))
        assert torch.equal(a, ops.embed_wgrad(gy, ids.int(), V))


def test_wgrad_strided_and_broadcast_gradients():
    ids = make_ids(600, 9, "padded", 1).view(20, 30)
    big = torch.randn(20, 30, 150, device=DEV)
    for gy in (big[..., 5:101], big[..., ::3], torch.ones((), device=DEV).expand(20, 30, 64),
               torch.randn(30, 20, 40, device=DEV).transpose(0, 1), torch.randn(20, 1, 40, device=DEV).expand(20, 30, 40)):
        check_wgrad(ops.embed_wgrad(gy, ids, 9), gy, ids, 9, 1.0, F32)
    assert ops.embed_wgrad(big[..., :0], ids, 9).shape == (9, 0)
    empty = ops.embed_wgrad(big[:0], ids[:0], 9, dtype=BF16)
    assert empty.shape == (9, 150) and bool((empty == 0).all())


def test_wgrad_keeps_infinities_and_nans_to_their_tokens():
    """A masked position's gradient is not read into any sum, whatever it holds; a NaN stays with its own token."""
    for V in (4, 900):
        gy = torch.ones(64, 40, device=DEV)
        ids = torch.arange(64, device=DEV) % 4
        ids[5], gy[5] = -1, float("nan")
        ids[6], gy[6] = V, float("inf")
        gy[8, 3] = float("nan")                                # token 0
        gy[9, 4] = float("inf")                                # token 1
        dw = ops.embed_wgrad(gy, ids, V)
        assert bool(dw[0, 3].isnan()) and bool(dw[1, 4] == float("inf"))
        dw[0, 3] = dw[1, 4] = 16.0
        want = torch.zeros(V, 40, device=DEV)
        want[:4] = torch.tensor([16.0, 15.0, 15.0, 16.0], device=DEV)[:, None]
        want[1, 4] = 16.0
        assert torch.equal(dw, want)


def test_buffers_beside_the_outputs_stay_as_they_were():
    """The C entry points on outputs and a workspace inside larger buffers, at their smallest alignment."""
    L = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    for n, V, C, off in ((777, 5, 33, 1), (777, 5, 64, 4), (2000, 321, 64, 3), (5, 1000, 24, 4)):
        ids = make_ids(n, V, "padded", n)
        w = torch.randn(V, C, device=DEV)
        ybuf = torch.full((n * C + 64,), 7.0, device=DEV)
        y = ybuf[off:off + n * C]
        _lib.check(L.bpc_embed_lookup(ids.data_ptr(), 8, w.data_ptr(), y.data_ptr(), n, V, C, C, 2.0, 0, 0, st), "lookup")
        check_lookup(y.view(n, C), ids, w, 2.0, F32)
        assert bool((ybuf[:off] == 7).all()) and bool((ybuf[off + n * C:] == 7).all())
        gbuf = torch.randn(n * C + 8, device=DEV)
        gy = gbuf[off:off + n * C].view(n, C)
        dbuf = torch.full((V * C + 64,), 7.0, device=DEV)
        dw = dbuf[off:off + V * C]
        need = int(L.bpc_embed_wgrad_workspace_size(n, V, C))
        ws = torch.full((need + 4096,), 5, device=DEV, dtype=torch.uint8)
        _lib.check(L.bpc_embed_wgrad(gy.data_ptr(), ids.data_ptr(), 8, dw.data_ptr(), ws.data_ptr(), need, n, V, C, C,
                                     1.0, 0, 0, st), "wgrad")
        check_wgrad(dw.view(V, C), gy, ids, V, 1.0, F32)
        assert bool((dbuf[:off] == 7).all()) and bool((dbuf[off + V * C:] == 7).all()) and bool((ws[need:] == 5).all())


def test_embedding_gradients_by_autograd_and_differences():
    """The autograd function against nn.functional.embedding, and its gradient against central differences of a
    quadratic loss (whose differences have no error of their own but fp32's)."""
    w = torch.randn(11, 24, device=DEV, requires_grad=True)
    ids = make_ids(90, 11, "padded", 2).view(9, 10)
    t = torch.randn(9, 10, 24, device=DEV)
    loss = lambda v: (ops.embedding(ids, v, 0.5) * t).sum() + 0.5 * (ops.embedding(ids, v, 0.5) ** 2).sum()
    g, = torch.autograd.grad(loss(w), w)
    ok = ((ids >= 0) & (ids < 11))[..., None]
    w64 = w.detach().double().requires_grad_()
    e = 0.5 * w64[ids.clamp(0, 10)] * ok
    g64, = torch.autograd.grad((e * t.double()).sum() + 0.5 * (e ** 2).sum(), w64)
    assert float((g - g64).abs().max()) < 1e-5 * float(g64.abs().max())
    d = torch.randn_like(w)
    with torch.no_grad():
        num = (loss((w + 0.25 * d)).double() - loss((w - 0.25 * d)).double()) / 0.5
    scale = float((t.abs().sum() + 90 * 24 * 10))               # what the loss's fp32 sums round against
    assert abs(float(num) - float((g64 * d).sum())) < 64 * 2.0**-24 * scale
    # types: a bf16 table gets a bf16 gradient, whatever the output's type
    wb = w.detach().to(BF16).requires_grad_()
    y = ops.embedding(ids, wb, dtype=F32)
    y.sum().backward()                                          # a broadcast gradient
    assert y.dtype == F32 and wb.grad.dtype == BF16
    m = torch.bincount(ids[(ids >= 0) & (ids < 11)], minlength=11)
    assert torch.equal(wb.grad, m[:, None].expand(11, 24).to(BF16))
    # an unused output, a table without a gradient, a second derivative
    assert not ops.embedding(ids, w.detach()).requires_grad
    y = ops.embedding(ids, w)
    g1, = torch.autograd.grad((y ** 2).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g1.sum(), w)
    # ids changed between the passes: autograd notices
    mine = ids.clone()
    y = ops.embedding(mine, w)
    mine.zero_()
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_other_streams_and_captured_replays():
    """A call on a side stream, and forward + gradient replayed from two graphs with new inputs in each replay."""
    V, C, n = 200, 64, 5000
    w = torch.randn(V, C, device=DEV)
    ids, gy = make_ids(n, V, "hot", 1), torch.randn(n, C, device=DEV)
    want = ops.embed_wgrad(gy, ids, V)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.embed_wgrad(gy, ids, V)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for Vk in (V, 3):
        i, x = (ids % Vk).clone(), gy.clone()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, dw = ops.embed_lookup(i, w), ops.embed_wgrad(x, i, Vk)
        graphs.append((g, i, x, y, dw, Vk))
    for seed in (4, 5):
        for g, i, x, y, dw, Vk in graphs:
            i.copy_(make_ids(n, Vk, "padded", seed))
            x.copy_(torch.randn(n, C, device=DEV))
        for g, *_ in graphs:
            g.replay()
        for g, i, x, y, dw, Vk in graphs:
            assert torch.equal(dw, ops.embed_wgrad(x, i, Vk)) and torch.equal(y, ops.embed_lookup(i, w))


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    w, ids = torch.randn(9, 40, device="cuda:1"), torch.randint(0, 9, (70,), device="cuda:1")
    with torch.cuda.device(0):
        y = ops.embed_lookup(ids, w)
        dw = ops.embed_wgrad(y, ids, 9)
    assert y.device == dw.device == w.device and torch.equal(y, w[ids])
    check_wgrad(dw, y, ids, 9, 1.0, F32)


def test_refusals():
    w, ids = torch.randn(9, 40, device=DEV), torch.randint(0, 9, (7,), device=DEV)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.embed_lookup(ids.short(), w)
    with pytest.raises(TypeError, match="int32 or int64"):
        ops.embed_lookup(ids.float(), w)
    with pytest.raises(TypeError, match="fp32"):
        ops.embed_lookup(ids, w.double())
    with pytest.raises(TypeError, match="fp32"):
        ops.embed_lookup(ids, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="V, C"):
        ops.embed_lookup(ids, w[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embed_lookup(ids.cpu(), w)
    gy = torch.randn(7, 40, device=DEV)
    with pytest.raises(ValueError, match="shape"):
        ops.embed_wgrad(gy[:6], ids, 9)
    with pytest.raises(ValueError, match="shape"):
        ops.embed_wgrad(gy.view(7, 4, 10), ids, 9)
    with pytest.raises(TypeError, match="fp32"):
        ops.embed_wgrad(gy.double(), ids, 9)
    with pytest.raises(ValueError, match="tokens"):
        ops.embed_wgrad(gy, ids, 0)
