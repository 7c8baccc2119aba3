"""Linear attention with a decay for each head on the GPU (whole sequences, gradients, single positions) against its
definition in 64 bits.

Tolerances, u = 2^-24.  Every output is a sum of products weighed by powers of the decay: with every factor replaced by its
magnitude the same sum gives mag.  The sums over D elements of a head and over T positions, and the state's updates, each
round once; a power a^n is off by (n + 4) u of itself: together at most (D + 4 T) u mag.  fp32 products are made of
operands in two tf32 parts of 11 bits: what the second part rounds away is 2^-23 of the operand, twice, and the product
of the second parts, left out, 2^-22: 8 u a product, and an element is a product of products, of the state with the rows
and of the rows that made it: 3 of them, and 8 u for the powers' and the scale's: 48 u mag at most with the sums' ends.
For bf16 inputs, products of the inputs are exact; an fp32 factor (the weighted pair, the state, the weighted row in it) goes
in as two bf16 parts, off by (2^-9)^2 = 64 u of itself, at most two such factors in a term of a bf16 result: 128 u mag.
A state handed out has its rows in three parts.  Then the rounding to the type: half a step.  That is a
bound for the worst case.  Against a loss of bits the root mean square is tested too, over results of a thousand values and
more (n = (sum v^2)^2 / sum v^4 counts them): roundings to the type are spread evenly over half a step either way, so
their squares are a third of its square on average, with a deviation of 0.3 / sqrt(n), of which six are allowed; a single
value may be off by the whole half step, so fewer values say nothing.  fp32 results, whose T + D roundings are independent,
are off by about u sqrt(T + D) / sqrt(3) of the root mean square, of which 8 u sqrt(T + D) is allowed."""
import pytest
import torch

from codecoder_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0**-24
HALF = {F32: 2.0**-24, BF16: 2.0**-8}


def decays(H, lo=1.0, hi=8.0):
    return torch.log1p(-torch.exp2(-torch.linspace(lo, hi, H, device=DEV, dtype=torch.float64))).float()


def make(B, T, H, dk, dv, dtype, seed, state=False, lengths=None):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dt=dtype):
        return torch.randn(*shape, generator=g, device=DEV).to(dt)
    s = dict(q=normal(B, T, H, dk), k=normal(B, T, H, dk), v=normal(B, T, H, dv), go=normal(B, T, H, dv),
             g=decays(H), s0=normal(B, H, dk, dv, dt=F32) if state else None,
             gs=normal(B, H, dk, dv, dt=F32) if state else None, n=None)
    if lengths is not None:
        s["n"] = torch.as_tensor(lengths, device=DEV)
    return s


def definition(q, k, v, g, scale, s0, n, go=None, gs=None, mag=False):
    """The recurrence and its gradients, position by position in 64 bits."""
    q, k, v, go, s0, gs = (None if t is None else t.double().abs() if mag else t.double() for t in (q, k, v, go, s0, gs))
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    a = torch.exp(g.double())[:, None, None]
    n = torch.full((B,), T, device=q.device) if n is None else n.long().clamp(0, T)
    S = q.new_zeros(B, H, dk, dv) if s0 is None else s0
    states, o = [S], torch.zeros_like(v)
    for t in range(T):
        live = (t < n)[:, None, None, None]
        kt = torch.where(live[..., 0], k[:, t], 0)
        vt = torch.where(live[..., 0], v[:, t], 0)
        qt = torch.where(live[..., 0], q[:, t], 0)
        S = torch.where(live, a * S + kt[..., :, None] * vt[..., None, :], S)
        states.append(S)
        o[:, t] = scale * (qt[..., None, :] @ S)[..., 0, :] * live[..., 0]
    if go is None:
        return o, S
    dS = torch.zeros_like(S) if gs is None else gs
    dq, dk_, dv_ = (torch.zeros_like(t) for t in (q, k, v))
    for t in reversed(range(T)):
        live = (t < n)[:, None, None, None]
        z = live[..., 0]
        qt, kt, vt, gt = (torch.where(z, x[:, t], 0) for x in (q, k, v, go))
        dq[:, t] = scale * (states[t + 1] @ gt[..., None])[..., 0] * z
        dS = torch.where(live, dS + scale * qt[..., :, None] * gt[..., None, :], dS)
        dk_[:, t] = (dS @ vt[..., None])[..., 0] * z
        dv_[:, t] = (kt[..., None, :] @ dS)[..., 0, :] * z
        dS = torch.where(live, a * dS, dS)
    return o, S, dq, dk_, dv_, dS


def check(got, want, mag, dtype, T, D, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    e = (D + 4 * T + 48 + (128 if dtype == BF16 else 0)) * U * mag
    tol = e + (want.abs() + e) * HALF[dtype] + 1e-36
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (what, float((err / tol).max()))
    sq = want.square()
    n = float(sq.sum()**2 / sq.square().sum()) if want.numel() and bool((sq > 0).any()) else 0.0
    if n >= 1000:
        bound = (HALF[dtype] * (1 / 3 + 1.8 / n**0.5)**0.5 if dtype != F32 else 0.0) + 8 * U * (T + D)**0.5
        got_rms = float((err.square().mean() / sq.mean()).sqrt())
        assert got_rms <= bound, (what, "rms", got_rms, bound)


def run(s, scale=None, need=("q", "k", "v", "s0")):
    q, k, v, g, s0, n, go, gs = (s[x] for x in ("q", "k", "v", "g", "s0", "n", "go", "gs"))
    B, T, H, dk = q.shape
    dv, dtype = v.shape[-1], q.dtype
    sc = dk**-0.5 if scale is None else scale
    want = definition(q, k, v, g, sc, s0, n, go, gs)
    mag = definition(q, k, v, g, abs(sc), s0, n, go, gs, mag=True)
    D = max(dk, dv)
    o, S = ops.linear_attention(q, k, v, g, scale, s0, n, return_state=True)
    check(o, want[0], mag[0], dtype, T, D, "o")
    check(S, want[1], mag[1], F32, T, D, "state")
    check(ops.linear_attention(q, k, v, g, scale, s0, n), want[0], mag[0], dtype, T, D, "o alone")
    leaves = {x: s[x].detach().requires_grad_() for x in need if s[x] is not None}
    a = {**s, **leaves}
    o, S = ops.linear_attention(a["q"], a["k"], a["v"], g, scale, a["s0"], n, return_state=True)
    outs, gouts = ([o, S], [go, gs]) if gs is not None else ([o], [go])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gouts)))
    for name, i in (("q", 2), ("k", 3), ("v", 4), ("s0", 5)):
        if name in grads:
            check(grads[name], want[i], mag[i], F32 if name == "s0" else dtype, T, D, "d" + name)
    return o.detach(), S.detach(), grads


SHAPES = [(1, 1, 1, 1, 1), (2, 1, 3, 32, 32), (3, 5, 25, 32, 32), (4, 11, 7, 32, 32), (2, 15, 5, 64, 64), (2, 16, 2, 16, 16),
          (2, 17, 3, 32, 32), (2, 31, 3, 24, 40), (1, 33, 2, 40, 24), (2, 64, 2, 128, 128), (2, 65, 2, 64, 64),
          (1, 100, 3, 13, 7), (1, 127, 2, 128, 16), (1, 129, 1, 16, 128), (2, 200, 4, 32, 32), (1, 333, 5, 24, 40),
          (3, 257, 2, 96, 96), (700, 11, 4, 32, 32)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients_match_the_definition(shape, dtype):
    k = SHAPES.index(shape)
    run(make(*shape, dtype, k, state=False))
    run(make(*shape, dtype, k, state=True), scale=[0.3, -2.0, 1.0][k % 3])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [2, 3, 7, 8, 9, 15, 16, 17, 32])
def test_lengths_where_the_kernels_change(T, dtype):
    for D in (8, 16, 24, 32, 40, 64):
        run(make(3, T, 5, D, D, dtype, T + D))
    run(make(3, T, 5, 24, 32, dtype, T, lengths=[T, T - 1, 1]))
    run(make(2, T, 3, 64, 16, dtype, T, state=True))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,dk,dv", [(11, 32, 32), (40, 64, 64), (150, 24, 40), (300, 32, 32)])
def test_lengths(T, dk, dv, dtype):
    lengths = [0, 1, T, T // 2, T - 1, T + 5, -3, min(16, T), min(17, T)]
    for state in (False, True):
        for it in (torch.int32, torch.int64):
            s = make(len(lengths), T, 3, dk, dv, dtype, T, state, torch.tensor(lengths, dtype=it))
            ref, S, grads = run(s)
    # what lies behind a sequence's length is not read, whatever it is
    dead = (torch.arange(T, device=DEV) >= s["n"].clamp(0, T)[:, None])[:, :, None, None]
    bad = {**s, **{x: torch.where(dead, torch.full_like(s[x], v), s[x])
                   for x, v in (("q", float("nan")), ("k", float("inf")), ("v", -float("inf")), ("go", float("nan")))}}
    o, S2 = ops.linear_attention(bad["q"], bad["k"], bad["v"], s["g"], None, s["s0"], s["n"], return_state=True)
    assert torch.equal(o, ref) and torch.equal(S2, S) and bool((o[dead.expand_as(o)] == 0).all())
    leaves = [bad[x].requires_grad_() for x in ("q", "k", "v", "s0")]
    got = ops.linear_attention(*leaves[:3], s["g"], None, leaves[3], s["n"], return_state=True)
    for x, g in zip(("q", "k", "v", "s0"), torch.autograd.grad(got, leaves, (bad["go"], s["gs"]))):
        assert torch.equal(g, grads[x])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays_at_the_ends(dtype):
    for T in (9, 50, 140):
        s = make(2, T, 5, 32, 32, dtype, T, True)
        s["g"] = torch.tensor([0.0, -float("inf"), -100.0, -1e-4, -0.7], device=DEV)
        run(s)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,H,D", [(1, 2500, 2, 64), (2, 1100, 3, 32), (1, 1500, 1, 128), (1, 2049, 2, 20)])
def test_long_sequences(B, T, H, D, dtype):
    s = make(B, T, H, D, D, dtype, T, True)
    s["g"] = decays(H, 3.0, 10.0)
    run(s)
    s["n"] = torch.tensor([T - 700, 3][:B], device=DEV)
    run(s)


@pytest.mark.parametrize("with_state", [False, True])
def test_offsets_past_32_bits(with_state):
    """Rows more than 2^31 elements apart, and a sequence's positions too; without a state in registers, with one in chunks."""
    B, T, H, D = 2, 3, 2, 32
    s = make(B, T, H, D, D, BF16, 3, with_state)
    far = {}
    for i, x in enumerate(("q", "k", "v", "go")):
        wide = torch.empty((B - 1) * 6 * 2**29 + (T - 1) * 2**30 + H * D, device=DEV, dtype=BF16)
        far[x] = wide.as_strided((B, T, H, D), (6 * 2**29, 2**30, D, 1))
        far[x].copy_(s[x])
    ref = ops.linear_attention(s["q"], s["k"], s["v"], s["g"], state=s["s0"])
    leaves = [far[x].requires_grad_() for x in "qkv"]
    o = ops.linear_attention(*leaves, s["g"], state=s["s0"])
    assert torch.equal(o, ref)
    grads = torch.autograd.grad(o, leaves, far["go"])
    near = [s[x].requires_grad_() for x in "qkv"]
    for p, q in zip(grads, torch.autograd.grad(ops.linear_attention(*near, s["g"], state=s["s0"]), near, s["go"])):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_gradients_do_not_need_the_forwards_workspace(dtype):
    """bpc_linear_attention_bwd with and without the workspace that the forward pass left, over several segments."""
    from array import array

    from codecoder_b200 import _lib
    B, T, H, dk, dv = 2, 700, 2, 32, 24
    s = make(B, T, H, dk, dv, dtype, 6, True)
    s["n"] = torch.tensor([650, 90], device=DEV)
    L, code = _lib.lib(), _lib.BPC_DTYPE_F32 if dtype == F32 else _lib.BPC_DTYPE_BF16
    tensors = [s[x] for x in ("q", "k", "v", "go")]
    strides = array("q", [st for t in tensors for st in t.stride()[:3]])
    at = strides.buffer_info()[0]
    fwd_ws, bwd_ws = (torch.empty(int(L.bpc_linear_attention_workspace_size(B, T, H, dk, dv, code, i)), device=DEV, dtype=torch.uint8)
                      for i in range(2))
    assert fwd_ws.numel() > 16                      # several segments
    o, end = torch.empty_like(s["v"]), torch.empty_like(s["s0"])
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: None if t is None else t.data_ptr()
    _lib.check(L.bpc_linear_attention_fwd(p(s["q"]), p(s["k"]), p(s["v"]), p(o), p(s["g"]), p(s["s0"]), p(end), p(s["n"]), 8, B, T, H,
                                          dk, dv, at, 0.5, code, p(fwd_ws), fwd_ws.numel(), stream), "fwd")
    out = []
    for ws in (fwd_ws, None):
        g = [torch.empty_like(s[x]) for x in ("q", "k", "v", "s0")]
        _lib.check(L.bpc_linear_attention_bwd(*(p(t) for t in tensors), p(s["g"]), p(s["s0"]), p(s["gs"]), p(ws), p(s["n"]), 8,
                                              *(p(t) for t in g), B, T, H, dk, dv, at, 0.5, code, p(bwd_ws), bwd_ws.numel(), stream),
                   "bwd")
        out.append(g)
    want = definition(*(s[x] for x in "qkv"), s["g"], 0.5, s["s0"], s["n"], s["go"], s["gs"])
    mag = definition(*(s[x] for x in "qkv"), s["g"], 0.5, s["s0"], s["n"], s["go"], s["gs"], mag=True)
    check(o, want[0], mag[0], dtype, T, 32, "o")
    for g in out:
        for name, t, i in zip(("q", "k", "v", "s0"), g, range(2, 6)):
            check(t, want[i], mag[i], F32 if name == "s0" else dtype, T, 32, "d" + name)


def test_two_streams_at_once():
    """Calls on two streams, each with its own workspaces, do not disturb one another."""
    cases = [make(2, 900, 2, 64, 64, BF16, i, True) for i in range(2)]
    call = lambda s: ops.linear_attention(s["q"], s["k"], s["v"], s["g"], state=s["s0"], return_state=True)
    want = [call(s) for s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, end in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(end, want[i][1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype):
    B, T, H, D = 3, 37, 4, 32
    base = make(B, T, H, D, D, dtype, 8, True)

    def packed(t):                 # heads of a wider row, at an odd offset
        wide = torch.full((B, T, 3 * H * D + 1), float("nan"), device=DEV, dtype=dtype)
        wide[..., 1:1 + H * D] = t.reshape(B, T, H * D)
        return wide[..., 1:1 + H * D].unflatten(2, (H, D))

    def aligned(t):
        wide = torch.full((B, T, 3, H, D), float("nan"), device=DEV, dtype=dtype)
        wide[:, :, 1] = t
        return wide[:, :, 1]

    def heads_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def broken(t):                 # elements of a head not next to one another
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    ref = None
    for view in (lambda t: t, packed, aligned, heads_first, broken):
        s = {**base, **{x: view(base[x]) for x in ("q", "k", "v", "go")}}
        out = run(s)
        if ref is not None:
            assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
            assert all(torch.equal(out[2][x], ref[2][x]) for x in ref[2])
        ref = out
    # shared heads: one key for all of them, its gradient summed by autograd
    k = base["k"][:, :, :1].clone().requires_grad_()
    o = ops.linear_attention(base["q"], k.expand(B, T, H, D), base["v"], base["g"])
    dk, = torch.autograd.grad(o, k, base["go"])
    full = base["k"][:, :, :1].expand(B, T, H, D).contiguous().requires_grad_()
    want, = torch.autograd.grad(ops.linear_attention(base["q"], full, base["v"], base["g"]), full, base["go"])
    assert torch.equal(dk, want.sum(2, keepdim=True))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (2, 578, 32, 32), (3, 5, 24, 40), (1, 7, 128, 128), (5, 3, 13, 7),
                                       (64, 20, 16, 16), (2, 3, 64, 96), (1, 2, 100, 4)])
def test_steps_go_on_where_a_sequence_ends(B, H, dk, dv, dtype):
    T, more = 7, 3
    s = make(B, T + more, H, dk, dv, dtype, B + H, True)
    want_o, want_S = definition(s["q"], s["k"], s["v"], s["g"], dk**-0.5, s["s0"], None)
    mag_o, mag_S = definition(s["q"], s["k"], s["v"], s["g"], dk**-0.5, s["s0"], None, mag=True)
    _, S = ops.linear_attention(s["q"][:, :T], s["k"][:, :T], s["v"][:, :T], s["g"], state=s["s0"], return_state=True)
    other = torch.empty_like(S)
    for t in range(T, T + more):
        before = S.clone()
        o2 = ops.linear_attention_step(s["q"][:, t], s["k"][:, t], s["v"][:, t], s["g"], S, new_state=other)
        assert torch.equal(S, before)
        o = ops.linear_attention_step(s["q"][:, t], s["k"][:, t], s["v"][:, t], s["g"], S)
        assert torch.equal(o, o2) and torch.equal(S, other)
        check(o, want_o[:, t], mag_o[:, t], dtype, T + more, max(dk, dv), "step")
    check(S, want_S, mag_S, F32, T + more, max(dk, dv), "state")


def test_empty_calls():
    g = decays(3)
    for B, T, H in ((0, 5, 3), (2, 0, 3), (2, 4, 0)):
        q = torch.zeros(B, T, H, 16, device=DEV, requires_grad=True)
        s0 = torch.randn(B, H, 16, 16, device=DEV, requires_grad=True)
        o, S = ops.linear_attention(q, q, q, g[:H], state=s0, return_state=True)
        assert o.shape == q.shape and torch.equal(S, s0)
        dq, ds = torch.autograd.grad([o, S], [q, s0], [torch.zeros_like(o), torch.ones_like(S)])
        assert dq.shape == q.shape and bool((ds == 1).all())
        _, S = ops.linear_attention(q.detach(), q.detach(), q.detach(), g[:H], return_state=True)
        assert bool((S == 0).all())
    e = torch.zeros(0, 3, 16, device=DEV)
    assert ops.linear_attention_step(e, e, e, g, torch.zeros(0, 3, 16, 16, device=DEV)).shape == (0, 3, 16)


def test_gradients_match_differences():
    torch.manual_seed(9)
    B, T, H, D = 2, 21, 2, 8
    names = ("q", "k", "v", "s0")
    x = {n: torch.randn(*((B, H, D, D) if n == "s0" else (B, T, H, D)), device=DEV, dtype=torch.float64) for n in names}
    d = {n: torch.randn_like(x[n]) for n in names}
    go, gs = torch.randn(B, T, H, D, device=DEV), torch.randn(B, H, D, D, device=DEV)
    g = decays(H)

    def loss(e):
        o, S = definition(x["q"] + e * d["q"], x["k"] + e * d["k"], x["v"] + e * d["v"], g, 0.5, x["s0"] + e * d["s0"], None)
        return float((o * go.double()).sum() + (S * gs.double()).sum())
    h = 1e-5
    diff = (loss(h) - loss(-h)) / (2 * h)
    leaves = [x[n].float().requires_grad_() for n in names]
    out = ops.linear_attention(*leaves[:3], g, 0.5, leaves[3], return_state=True)
    grads = torch.autograd.grad(out, leaves, (go, gs))
    got = sum(float((t.double() * d[n]).sum()) for n, t in zip(names, grads))
    size = sum(float((t.double() * d[n]).abs().sum()) for n, t in zip(names, grads))
    assert abs(got - diff) <= 1e-5 * size, (got, diff, size)      # inputs rounded to fp32: u of every term and factor


def test_one_sided_gradients():
    s = make(2, 20, 3, 32, 32, F32, 4, True)
    leaves = [s[x].requires_grad_() for x in ("q", "k", "v", "s0")]
    want = definition(*(s[x] for x in "qkv"), s["g"], 32**-0.5, s["s0"], None, torch.zeros_like(s["go"]), s["gs"])
    o, S = ops.linear_attention(*leaves[:3], s["g"], state=leaves[3], return_state=True)
    for got, ref in zip(torch.autograd.grad(S, leaves, s["gs"], retain_graph=True), want[2:]):
        assert float((got.double() - ref.detach()).abs().max()) <= 1e-4 * float(ref.detach().abs().max()) + 1e-30
    only_o = torch.autograd.grad(o, leaves, s["go"])
    again = torch.autograd.grad(ops.linear_attention(*leaves[:3], s["g"], state=leaves[3]), leaves, s["go"])
    for p, r in zip(only_o, definition(*(s[x] for x in "qkv"), s["g"], 32**-0.5, s["s0"], None, s["go"])[2:]):
        assert float((p.double() - r.detach()).abs().max()) <= 1e-4 * float(r.detach().abs().max())
    assert all(torch.equal(p, q) for p, q in zip(only_o, again))


@pytest.mark.parametrize("shape", [(30, 11, 6, 32, 32), (2, 1500, 2, 64, 64)])
def test_repeats_bit_for_bit_on_any_stream_and_from_graphs(shape):
    s = make(*shape, BF16, 2, True)
    leaves = [s[x].requires_grad_() for x in ("q", "k", "v", "s0")]

    def once():
        out = ops.linear_attention(*leaves[:3], s["g"], state=leaves[3], return_state=True)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (s["go"], s["gs"])))
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
        for t in leaves:
            t.mul_(0.5)
    second = once()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(p, q) for p, q in zip(out, second))


def test_refusals():
    s = make(2, 6, 3, 16, 16, F32, 1, True)
    q, k, v, g, s0 = (s[x] for x in ("q", "k", "v", "g", "s0"))
    f, step = ops.linear_attention, ops.linear_attention_step
    with pytest.raises(ValueError, match="log_decay"):
        f(q, k, v, g[:2])
    with pytest.raises(ValueError, match="gradient"):
        f(q, k, v, g.clone().requires_grad_())
    with pytest.raises(TypeError, match="log_decay"):
        f(q, k, v, g.double())
    with pytest.raises(TypeError, match="one type"):
        f(q, k, v.bfloat16(), g)
    with pytest.raises(TypeError, match="fp32 or bf16"):
        f(q.half(), k.half(), v.half(), g)
    with pytest.raises(ValueError, match="shape"):
        f(q, k[:, :5], v, g)
    with pytest.raises(ValueError, match="shape"):
        f(q, k, v[:, :, :2], g)
    with pytest.raises(ValueError, match="head sizes"):
        f(torch.zeros(1, 2, 3, 129, device=DEV), torch.zeros(1, 2, 3, 129, device=DEV), v[:1, :2], g)
    with pytest.raises(ValueError, match="state"):
        f(q, k, v, g, state=s0[:1])
    with pytest.raises(TypeError, match="state"):
        f(q, k, v, g, state=s0.double())
    with pytest.raises(TypeError, match="lengths"):
        f(q, k, v, g, lengths=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="lengths"):
        f(q, k, v, g, lengths=torch.ones(3, device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="scale"):
        f(q, k, v, g, scale=float("nan"))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q, k.cpu(), v, g)
    with pytest.raises(ValueError, match="contiguous"):
        step(q[:, 0], k[:, 0], v[:, 0], g, s0.transpose(2, 3))
    with pytest.raises(ValueError, match="state must be"):
        step(q[:, 0], k[:, 0], v[:, 0], g, s0[:1])
    with pytest.raises(ValueError, match="gradient"):
        step(q[:, 0], k[:, 0], v[:, 0], g, s0.clone().requires_grad_())
    with pytest.raises(ValueError, match="dimensions"):
        step(q, k, v, g, s0)
    both = torch.zeros(3, 3, 16, 16, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        step(q[:, 0], k[:, 0], v[:, 0], g, both[:2], new_state=both[1:])


NAN_BITS = {F32: (0x7fc00000, 0x7fffffff, -1, 0x7f800001), BF16: (0x7fc0, 0x7fff, -1, 0x7f81)}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,at", [(1, 0), (5, 2), (12, 11), (16, 0), (40, 35), (100, 50), (700, 400)])
@pytest.mark.parametrize("where", ["q", "k", "v", "go", "s0"])
def test_values_that_are_not_finite_show(dtype, T, at, where):
    """NaN of any bits, and infinities, in one element: not finite where the definition is not, and finite 32 positions and
    more before (for o) or behind (for gradients) wherever the definition is."""
    ints = {F32: torch.int32, BF16: torch.int16}
    for n, bits in enumerate((*NAN_BITS[dtype], None)):
        s = make(2, T, 2, 24, 40, dtype, 7 * T + n, state=where == "s0")
        x = s[where]
        if bits is None:
            bad = torch.tensor(float("inf"), device=DEV, dtype=x.dtype)
        else:
            bits = NAN_BITS[x.dtype][n]
            bad = torch.tensor(bits, device=DEV, dtype=ints[x.dtype]).view(x.dtype)
        if where == "s0":
            x[1, 1, 3, 5] = bad
        else:
            x[1, at, 1, 3] = bad
        want = definition(s["q"], s["k"], s["v"], s["g"], 24**-0.5, s["s0"], None, s["go"], s["gs"])
        leaves = [s[i].detach().requires_grad_() for i in ("q", "k", "v", "s0") if s[i] is not None]
        o, S = ops.linear_attention(*leaves[:3], s["g"], None, leaves[3] if where == "s0" else None, return_state=True)
        outs, gouts = ([o, S], [s["go"], s["gs"]]) if where == "s0" else ([o], [s["go"]])
        grads = torch.autograd.grad(outs, leaves, gouts)
        alone = ops.linear_attention(s["q"], s["k"], s["v"], s["g"], None, s["s0"])
        far = (torch.arange(T, device=DEV) - at).abs()[:, None, None] >= 32
        for what, a, b in (("o", o, want[0]), ("alone", alone, want[0]), *zip(("dq", "dk", "dv"), grads, want[2:5])):
            lost = a.isfinite() & ~b.isfinite()
            assert not bool(lost.any()), (what, n, int(lost.sum()))
            spread = ~a.isfinite() & b.isfinite() & far
            assert not bool(spread.any()), (what, n, int(spread.sum()))
        assert not bool((S.isfinite() & ~want[1].isfinite()).any()), ("state", n)
        if where == "s0":
            assert not bool((grads[3].isfinite() & ~want[5].isfinite()).any()), ("dstate", n)

