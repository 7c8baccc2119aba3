"""The gradient norm and clipping on the GPU against their definitions in 64 bits.

Tolerances.  norm: squares and sums are fp64 (a relative error of n 2^-53 at most), the result rounds to fp32: 2^-24
relative.  clip: the factor rounds to fp32 (2^-24), the product to fp32 (2^-24) and to the output's type (half a step),
plus half of its smallest subnormal."""
import math

import pytest
import torch

from codecoder_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0**-24, BF16: 2.0**-8, F16: 2.0**-11}
SUB = {F32: 2.0**-150, BF16: 2.0**-134, F16: 2.0**-25}


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check_norm(got, ref):
    assert got.dtype == F32 and got.shape == () and got.is_cuda
    assert abs(float(got) - ref) <= ref * (2.0**-24 + 1e-12) + 2.0**-150, (float(got), ref)


def check_clip(outs, ins, norm, max_norm):
    coef = min(1.0, max_norm / (norm + 1e-6))
    for o, t in zip(outs, ins):
        ref = t.double() * coef
        tol = ref.abs() * (HALF[o.dtype] + 2.1 * 2.0**-24) + SUB[o.dtype]
        assert bool(((o.double() - ref).abs() <= tol).all())


def make(sizes, dtypes, seed, sigma=1.0, bucket=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if bucket:
        flat = (torch.randn(sum(sizes), generator=g, device=DEV) * sigma).to(dtypes[0])
        return list(flat.split(sizes))
    return [(torch.randn(s, generator=g, device=DEV) * sigma).to(dtypes[k % len(dtypes)]) for k, s in enumerate(sizes)]


LISTS = [[1], [0, 1, 0], [7], [4095], [4096], [4097], [8, 9, 15, 16, 17], [100000], [3, 50000, 1, 1, 70001, 2],
         [1 + 37 * k % 211 for k in range(31)], [1 + 37 * k % 2011 for k in range(33)], [5] * 199, [9] * 201,
         [1 + 131 * k % 5000 for k in range(999)], [3] * 1000, [1 + k % 7 for k in range(2501)], [5000011, 13, 2000003]]


@pytest.mark.parametrize("k", range(len(LISTS)))
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("bucket", [False, True])
def test_norm_and_clip_match_the_definition(k, dtypes, bucket):
    ts = make(LISTS[k], dtypes, k, 0.5, bucket)
    ref = norm64(ts)
    check_norm(ops.grad_norm(ts), ref)
    before = [t.clone() for t in ts]
    for limit in (0.25 * ref, 2.0 * ref + 1.0):
        for outs in ([torch.full_like(t, 7.0) for t in ts], [torch.full_like(t, 7.0, dtype=F32) for t in ts],
                     [torch.full_like(t, 7.0, dtype=BF16) for t in ts]):
            check_norm(ops.clip_grads(ts, limit, out=outs), ref)
            check_clip(outs, before, ref, limit)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check_norm(ops.clip_grads(ts, 2.0 * ref + 1.0), ref)        # in place and within the limit: unchanged
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    check_norm(ops.clip_grads(ts, 0.25 * ref), ref)
    check_clip(ts, before, ref, 0.25 * ref)


def test_outputs_at_every_offset_and_their_neighbours():
    """Inputs and outputs at unequal offsets from a 16-byte boundary; what lies between the outputs stays."""
    for it in (F32, BF16, F16):
        for ot in (F32, BF16, F16):
            src = (torch.randn(9000, device=DEV) * 3).to(it)
            for a, b in ((0, 0), (1, 0), (0, 1), (3, 5), (7, 2), (8, 4), (5, 5)):
                dst = torch.full((9000,), 7.0, device=DEV, dtype=ot)
                ts = [src[a:a + 4200], src[4300 + b:4300 + b + 77], src[5000 + a:5000 + a + 1]]
                outs = [dst[b:b + 4200], dst[4300 + a:4300 + a + 77], dst[5000 + b:5000 + b + 1]]
                ref = norm64(ts)
                check_norm(ops.clip_grads(ts, 1.0, out=outs), ref)
                check_clip(outs, ts, ref, 1.0)
                used = torch.zeros(9000, device=DEV, dtype=torch.bool)
                for lo, n in ((b, 4200), (4300 + a, 77), (5000 + b, 1)):
                    used[lo:lo + n] = True
                assert bool((dst[~used] == 7).all())


def test_extreme_values():
    big = torch.tensor([3e38, -3e38, 1e20], device=DEV)
    check_norm(ops.grad_norm([big[2:]]), norm64([big[2:]]))      # its square is beyond fp32
    assert float(ops.grad_norm([big])) == float("inf")            # beyond fp32 itself, but the factor is right
    out = torch.empty_like(big)
    ops.clip_grads([big], 1.0, out=[out])
    check_clip([out], [big], norm64([big]), 1.0)
    small = torch.full((1000,), 1e-30, device=DEV)                # squares below fp32's subnormals
    check_norm(ops.grad_norm([small]), norm64([small]))
    check_norm(ops.grad_norm([torch.full((3,), 1e-45, device=DEV)]), norm64([torch.full((3,), 1e-45, device=DEV)]))
    zero = torch.zeros(50, device=DEV)
    assert float(ops.clip_grads([zero], 1.0)) == 0.0 and bool((zero == 0).all())
    x = torch.randn(50, device=DEV)
    assert float(ops.clip_grads([x], 0.0)) > 0 and bool((x == 0).all())
    x = torch.randn(50, device=DEV)
    keep = x.clone()
    ops.clip_grads([x], float("inf"))
    assert torch.equal(x, keep)


def test_infinities_and_nans_do_as_torch_does():
    for bad in (float("inf"), float("nan"), -float("inf")):
        p = [torch.nn.Parameter(torch.zeros(300, device=DEV)), torch.nn.Parameter(torch.zeros(5, device=DEV))]
        q = [torch.nn.Parameter(torch.zeros(300, device=DEV)), torch.nn.Parameter(torch.zeros(5, device=DEV))]
        for a, b in zip(p, q):
            a.grad = torch.randn_like(a)
            b.grad = a.grad.clone()
        p[0].grad[77] = q[0].grad[77] = bad
        a, b = ops.clip_grad_norm_(p, 1.0), torch.nn.utils.clip_grad_norm_(q, 1.0)
        assert torch.equal(a.isnan(), b.isnan()) and (bool(a.isnan()) or float(a) == float(b))
        for u, v in zip(p, q):
            assert torch.equal(u.grad.isnan(), v.grad.isnan()) and torch.equal(u.grad.nan_to_num(), v.grad.nan_to_num())


def test_clip_grad_norm_takes_what_torchs_does():
    net = torch.nn.Sequential(torch.nn.Linear(30, 70), torch.nn.Linear(70, 3)).to(DEV)
    twin = torch.nn.Sequential(torch.nn.Linear(30, 70), torch.nn.Linear(70, 3)).to(DEV)
    twin.load_state_dict(net.state_dict())
    x = torch.randn(40, 30, device=DEV)
    for m in (net, twin):
        m(x).square().sum().backward()
    net[1].bias.grad = twin[1].bias.grad = None                    # one without a gradient
    raw = [p.grad.clone() for p in net.parameters() if p.grad is not None]
    got, want = ops.clip_grad_norm_(net.parameters(), 0.5), torch.nn.utils.clip_grad_norm_(twin.parameters(), 0.5)
    check_norm(got, norm64(raw))
    assert abs(float(got) - float(want)) < 1e-5 * float(want)
    check_clip([p.grad for p in net.parameters() if p.grad is not None], raw, norm64(raw), 0.5)
    check_norm(ops.clip_grad_norm_(net[0].weight, 100.0), norm64([net[0].weight.grad]))
    assert float(ops.clip_grad_norm_([net[1].bias], 1.0)) == 0.0


def test_dense_tensors_in_any_order_of_dimensions():
    a = torch.randn(30, 40, device=DEV).t()
    b = torch.randn(3, 8, 5, 6, device=DEV).to(memory_format=torch.channels_last)
    ref, keep = norm64([a, b]), [a.clone(), b.clone()]
    outs = [torch.empty_strided(t.shape, t.stride(), device=DEV) for t in (a, b)]
    check_norm(ops.clip_grads([a, b], 1.0, out=outs), ref)
    check_clip(outs, keep, ref, 1.0)
    check_norm(ops.clip_grads([a, b], 1.0), ref)
    check_clip([a, b], keep, ref, 1.0)


def test_refusals():
    x = torch.randn(40, 50, device=DEV)
    with pytest.raises(ValueError, match="gaps or overlaps"):
        ops.grad_norm([x[:, :20]])
    with pytest.raises(ValueError, match="gaps or overlaps"):
        ops.clip_grads([x[:, :1].expand(40, 50)], 1.0)
    with pytest.raises(TypeError, match="takes dense"):
        ops.grad_norm([x, x.double()])
    with pytest.raises(ValueError, match="different devices"):
        ops.grad_norm([x, x.cpu()])
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grads([x, x], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.clip_grads([x, x[3]], 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.clip_grads([x], -1.0)
    with pytest.raises(ValueError, match="same shape"):
        ops.clip_grads([x], 1.0, out=[x.view(-1)])
    with pytest.raises(ValueError, match="same shape"):
        ops.clip_grads([x], 1.0, out=[])
    with pytest.raises(ValueError, match="strides"):
        ops.clip_grads([x], 1.0, out=[torch.empty(50, 40, device=DEV).t()])
    keep = x.clone()
    assert torch.equal(x, keep)
    check_norm(ops.grad_norm([x, x]), math.sqrt(2.0) * norm64([x]))       # the norm alone may read a tensor twice


def test_refused_clips_change_nothing():
    x = torch.randn(40, 50, device=DEV)
    keep, out = x.clone(), torch.full((40, 50), 7.0, device=DEV)
    for ts, limit, outs in (([x, x], 1.0, None), ([x, x[3]], 1.0, None), ([x], -1.0, None), ([x], float("nan"), None),
                            ([x, x.double()], 1.0, None), ([x, x[:, :20]], 1.0, None), ([x], 1.0, [x[:, :1].expand(40, 50)]),
                            ([x], 1.0, []), ([x], 1.0, [out.view(-1)]), ([x], 1.0, [torch.empty(50, 40, device=DEV).t()]),
                            ([x, keep], 1.0, [out, out]), ([x, keep], 1.0, [keep, out])):
        before = keep.clone()
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.clip_grads(ts, limit, out=outs)
        torch.cuda.synchronize()
        assert torch.equal(x, before) and torch.equal(keep, before) and bool((out == 7).all())


def test_autograd_notices_clipping_in_place():
    w = torch.randn(10, device=DEV, requires_grad=True)
    x = torch.randn(10, device=DEV)
    y = (w * x).sum()
    ops.clip_grads([x], 0.1)
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()
    with torch.inference_mode():
        z = torch.randn(10, device=DEV)
        assert float(ops.clip_grads([z], 0.1)) > 0.1


def test_repeats_side_streams_and_captured_replays():
    ts = make([1000, 77777, 3, 123456], (F32, BF16), 9)
    outs = [torch.empty_like(t) for t in ts]
    a = ops.clip_grads(ts, 1.0, out=outs)
    first = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ops.clip_grads(ts, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and all(torch.equal(o, f) for o, f in zip(outs, first))
    graphs = []
    for k in (2, 4):
        xs, os_ = [t.clone() for t in ts[:k]], [torch.empty_like(t) for t in ts[:k]]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norm = ops.clip_grads(xs, 1.0, out=os_)
        graphs.append((g, xs, os_, norm))
    for seed in (3, 4):
        for k, (g, xs, os_, norm) in enumerate(graphs):
            for x in xs:
                x.normal_(0, seed + k)
        for g, *_ in graphs:
            g.replay()
        for g, xs, os_, norm in graphs:
            check_norm(norm, norm64(xs))
            check_clip(os_, xs, norm64(xs), 1.0)


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x = torch.randn(5000, device="cuda:1")
    ref, keep = norm64([x]), x.clone()
    with torch.cuda.device(0):
        n = ops.clip_grads([x], 1.0)
    assert n.device == x.device
    check_clip([x], [keep], ref, 1.0)


def test_embedding_and_clipping_together():
    """A training step's pieces as they are used together: lookup, a loss, the deterministic gradient, clipping, against
    the same in 64 bits."""
    V, C = 50, 64
    w = torch.nn.Parameter(torch.randn(V, C, device=DEV))
    head = torch.nn.Parameter(torch.randn(C, 3, device=DEV))
    ids = torch.randint(-1, V, (16, 33), device=DEV)
    y = ops.embedding(ids, w, 2.0) @ head
    y.square().mean().backward()
    w64, h64 = w.detach().double().requires_grad_(), head.detach().double().requires_grad_()
    e = 2.0 * w64[ids.clamp_min(0)] * (ids >= 0)[..., None]
    (e @ h64).square().mean().backward()
    ref = norm64([w64.grad, h64.grad])
    got = ops.clip_grad_norm_([w, head], 0.1)
    coef = 0.1 / (ref + 1e-6)
    assert abs(float(got) - ref) < 1e-4 * ref                     # fp32 products of 64 and 528 terms
    for a, b in ((w, w64), (head, h64)):
        assert float((a.grad.double() - coef * b.grad).abs().max()) < 1e-4 * coef * float(b.grad.abs().max())
