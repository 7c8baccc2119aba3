"""Measured cases of the group-norm and linear-attention operators of codecoder_b200.ops.

  norm        y = act(w (x - mean) / sqrt(var + eps) + b), statistics per sample and group of channels,
              x (B, N, C) channels last                                                   ops.group_norm
  norm train  the same with the gradients of x, w and b                                   ops.group_norm, autograd
  memory      S_t = a_h S_(t-1) + k_t v_t^T, o_t = scale q_t S_t over t < length, a_h = exp(log_decay_h)
                                                                                          ops.linear_attention
  memory train  the same with the gradients of q, k, v and the first state                ops.linear_attention, autograd
  step        one t of it: the state of every head updated and read                       ops.linear_attention_step

`run` computes a case in its plain torch form, or, where `own` is true, by the library's calls; `exact` gives the
same outputs in 64 bits from the definitions."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
EPS = 1e-5
#: 512 BB72 shots of 504 nodes at 512 channels: no drawn case has more values
LARGEST = 512 * 504 * 512


def listed():
    return [
        # one BB72 shot in front of a block: latency
        dict(name="norm one shot", kind="norm", samples=1, rows=504, channels=512, groups=32, x="f32", y="bf16",
             act="silu", affine=True),
        # one group a sample, as a layer norm over a whole d = 13 shot's data nodes in fp32: no slice of it stands alone
        dict(name="norm whole shots", kind="norm", samples=64, rows=2197, channels=128, groups=1, x="f32", y="f32",
             act="gelu", affine=True),
        # a Cascade network's training batch of 512 BB72 shots: fp32 stream in, bf16 branch out, and back
        dict(name="norm cascade train", kind="norm train", samples=512, rows=504, channels=512, groups=32, x="f32",
             y="bf16", act="silu", affine=True),
        # the memory's output normalised head by head: 1,024 d = 11 shots, every data node a sample of its own
        dict(name="norm heads train", kind="norm train", samples=1024 * 11 * 121, rows=1, channels=96, groups=3,
             x="bf16", y="bf16", act="silu", affine=True),
        # odd everything: groups of 9 channels, which no vector width divides
        dict(name="norm odd train", kind="norm train", samples=37, rows=333, channels=45, groups=5, x="f16", y="f16",
             act="gelu", affine=True),
        # the d = 11 network's data stream (11 rounds x 121 sites x 3 heads of 32), 1,024 shots, forward and backward
        dict(name="memory d11 train", kind="memory train", batch=1024, length=11, heads=363, dk=32, dv=32, x="bf16",
             state=False, ragged=False),
        # the fp32 d = 5 network's shots: 5 rounds x 25 sites, one head of 32
        dict(name="memory d5 fp32", kind="memory", batch=1024, length=5, heads=25, dk=32, dv=32, x="f32",
             state=False, ragged=False),
        # two long experiments taken in at once before streaming goes on: few heads, many rounds, the state kept
        dict(name="memory long", kind="memory", batch=2, length=16384, heads=4, dk=64, dv=64, x="bf16", state=True,
             ragged=False),
        # training on one long run
        dict(name="memory long train", kind="memory train", batch=1, length=30011, heads=12, dk=64, dv=64, x="bf16",
             state=False, ragged=False),
        # odd everything: head sizes of 24 and 40, experiments of different lengths, a first state, fp32
        dict(name="memory odd train", kind="memory train", batch=9, length=333, heads=5, dk=24, dv=40, x="f32",
             state=True, ragged=True),
        # one round of one d = 17 stream: 289 sites x 2 heads of 32, latency
        dict(name="step one stream", kind="step", batch=1, heads=578, dk=32, dv=32, x="bf16"),
        # one round of 64 d = 13 streams: 169 sites x 4 heads of 32
        dict(name="step streams", kind="step", batch=64, heads=676, dk=32, dv=32, x="bf16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm train", "norm train", "memory", "memory train", "memory train", "step"])
    if kind.startswith("norm"):
        width = rng.choice([rng.randint(1, 24), 8 * rng.randint(1, 16)])
        groups = rng.choice([1, 2, 3, 4, 8, 32, rng.randint(1, 40)])
        channels = max(4, min(1024 // groups, width)) * groups
        rows = rng.choice([1, _spread(rng, 2, 3000), _spread(rng, 100, 3000)])
        samples = _spread(rng, 1, max(1, min(1500000, LARGEST // (2 * rows * channels))))
        x = rng.choice(["f32", "bf16", "bf16", "f16"])
        return dict(kind=kind, samples=samples, rows=rows, channels=channels, groups=groups, x=x,
                    y=rng.choice(["f32", "bf16"]) if x == "f32" else x, act=rng.choice(["none", "silu", "gelu"]),
                    affine=rng.random() < 0.8)
    dk, dv = rng.choice([(16, 16), (32, 32), (32, 32), (64, 64), (128, 128), (rng.randint(4, 128), rng.randint(4, 128))])
    if kind == "step":
        heads = _spread(rng, 1, 1200)
        return dict(kind=kind, batch=_spread(rng, 1, max(1, min(256, LARGEST // (4 * heads * dk * dv)))), heads=heads,
                    dk=dk, dv=dv, x=rng.choice(["bf16", "f32"]))
    length = rng.choice([_spread(rng, 1, 30), _spread(rng, 31, 1000), _spread(rng, 1001, 30000)])
    heads = _spread(rng, 1, max(1, min(1200, 4000000 // (length * max(dk, dv)))))
    batch = _spread(rng, 1, max(1, min(2000, LARGEST // (8 * length * heads * max(dk, dv)))))
    return dict(kind=kind, batch=batch, length=length, heads=heads, dk=dk, dv=dv, x=rng.choice(["bf16", "bf16", "f32"]),
                state=rng.random() < 0.4 and batch * heads * dk * dv < LARGEST // 8, ragged=rng.random() < 0.3)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    dt = DTYPES[case["x"]]

    def normal(*shape, dtype=dt, std=1.0):
        return torch.empty(*shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=g)

    if case["kind"].startswith("norm"):
        B, N, C = case["samples"], case["rows"], case["channels"]
        s["x"] = normal(B, N, C, std=1.5)
        s["x"] += normal(1, 1, C, std=0.5)              # a residual stream's channels have means of their own
        s["w"] = s["b"] = None
        if case["affine"]:
            s["w"] = 1 + normal(C, dtype=torch.float32, std=0.1)
            s["b"] = normal(C, dtype=torch.float32, std=0.1)
        if case["kind"] == "norm train":
            s["gy"] = normal(B, N, C, dtype=DTYPES[case["y"]], std=0.125)
            s["leaves"] = [t.requires_grad_() for t in (s["x"], s["w"], s["b"]) if t is not None]
        return s
    B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    # heads remember from two to about a thousand rounds
    s["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(1.0, 10.0, H, device=DEV, dtype=torch.float64))).float()
    s["scale"] = dk ** -0.5
    if case["kind"] == "step":
        s["q"], s["k"], s["v"] = normal(B, H, dk), normal(B, H, dk), normal(B, H, dv)
        s["state"] = normal(B, H, dk, dv, dtype=torch.float32)
        s["next"] = torch.empty_like(s["state"])        # a stream keeps two states and takes them in turn
        return s
    T = case["length"]
    s["q"], s["k"], s["v"] = normal(B, T, H, dk), normal(B, T, H, dk), normal(B, T, H, dv)
    s["s0"] = normal(B, H, dk, dv, dtype=torch.float32) if case["state"] else None
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    if case["kind"] == "memory train":
        s["go"] = normal(B, T, H, dv, std=0.125)
        s["gs"] = normal(B, H, dk, dv, dtype=torch.float32, std=0.125) if case["state"] else None
        s["leaves"] = [t.requires_grad_() for t in (s["q"], s["k"], s["v"], s["s0"]) if t is not None]
    return s


def _gate(z, act):
    """act(z) = z f and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        f = 1 / (1 + torch.exp(-z))
        return z * f, f * (1 + z * (1 - f))
    c = math.sqrt(2 / math.pi)
    f = 1 / (1 + torch.exp(-2 * c * (z + 0.044715 * z * z * z)))
    return z * f, f * (1 + z * (1 - f) * 2 * c * (1 + 3 * 0.044715 * z * z))


def _plain_norm(s):
    B, N, C, G = s["samples"], s["rows"], s["channels"], s["groups"]
    x = s["x"].detach().float().view(B, N, G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).mean((1, 3), keepdim=True) + EPS)
    xhat = xc * rstd
    w = 1.0 if s["w"] is None else s["w"].detach().view(G, C // G)
    z = xhat * w if s["b"] is None else xhat * w + s["b"].detach().view(G, C // G)
    y, dy = _gate(z, s["act"])
    y = y.view(B, N, C).to(DTYPES[s["y"]])
    if s["kind"] == "norm":
        return y
    gz = s["gy"].float().view(B, N, G, C // G) * dy
    a = gz * w
    dx = rstd * (a - a.mean((1, 3), keepdim=True) - xhat * (a * xhat).mean((1, 3), keepdim=True))
    dx = dx.view(B, N, C).to(s["x"].dtype)
    if s["w"] is None:
        return y, dx
    # sums over millions of rows: 64 bits
    dw = (gz * xhat).sum((0, 1), dtype=torch.float64).view(C).float()
    return y, dx, dw, gz.sum((0, 1), dtype=torch.float64).view(C).float()


def _plain_scan(a, b, c, g, x, last=None):
    """out_t = sum_(j <= t) e^(g (t - j)) (a_t . b_j) c_j + e^(g t) a_t x, (B, T, H, D) each and x (B, H, Da, Dc): chunks
    of 64, every chunk's part of the state and their weighted sums as products.  last (B) is each sequence's last t: also
    returns sum_j e^(g (last - j)) b_j c_j^T + e^(g last) x."""
    B, T, H, _ = a.shape
    L = min(64, T)
    n = -(-T // L)

    def cut(t):
        t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, n * L - T))
        return t.view(B, n, L, H, -1).permute(0, 3, 1, 2, 4)            # (B, H, n, L, D)

    a, b, c = cut(a), cut(b), cut(c)
    g = g.double()[:, None, None]
    i = torch.arange(L, device=DEV, dtype=torch.float64)

    def power(e):                                                       # e^(g e), zero where e < 0
        return torch.where(e >= 0, torch.exp(g * e.clamp_min(0)), 0.0).float()

    within = power(i[:, None] - i[None, :])                             # (H, L, L)
    out = ((a @ b.transpose(-1, -2)) * within[:, None]) @ c
    start = None
    if n > 1 or last is not None:
        # what chunk k adds to the state that the first t of chunk m sees: e^(g (L m - j)), j = L k + i
        part = (b * power(L - i)[:, 0, None, :, None]).transpose(-1, -2) @ c            # (B, H, n, Db, Dc)
        k = torch.arange(n, device=DEV, dtype=torch.float64)
        start = torch.einsum("hmk,bhkde->bhmde", power(L * (k[:, None] - 1 - k[None, :])), part)
    if x is not None:
        k = torch.arange(n, device=DEV, dtype=torch.float64)
        first = power(L * k)[:, 0, :, None, None] * x[:, :, None]
        start = first if start is None else start + first
    if start is not None:
        out = out + (a * power(i)[:, 0, None, :, None]) @ start
    out = out.permute(0, 2, 3, 1, 4).reshape(B, n * L, H, -1)[:, :T]
    if last is None:
        return out
    # the state as the last t's chunk leaves it
    m = (last.clamp_min(0) // L).view(B, 1, 1, 1, 1)
    r = (last - L * (last.clamp_min(0) // L)).double()
    e = r.view(B, 1, 1) - i.view(1, 1, L)
    weights = torch.where(e >= 0, torch.exp(g[None, :, 0] * e.clamp_min(0)), 0.0).float()      # (B, H, L)
    bm = torch.take_along_dim(b, m, 2)[:, :, 0] * weights[..., None]
    cm = torch.take_along_dim(c, m, 2)[:, :, 0]
    sm = torch.take_along_dim(start, m, 2)[:, :, 0]
    lead = torch.exp(g[:, 0, 0] * r.clamp_min(0)[:, None]).float()                  # (B, H)
    return out, bm.transpose(-1, -2) @ cm + lead[..., None, None] * sm


def _flip(t, lengths):
    """Each sequence's first lengths[b] entries in reverse order."""
    T = t.shape[1]
    at = lengths[:, None] - 1 - torch.arange(T, device=DEV)
    return torch.where((at >= 0)[:, :, None, None], torch.take_along_dim(t, at.clamp_min(0)[:, :, None, None], 1), 0)


def _plain_memory(s):
    q, k, v = (s[n].detach() for n in "qkv")
    B, T, H, dk = q.shape
    g, scale, s0 = s["log_decay"], s["scale"], s["s0"]
    n = torch.full((B,), T, device=DEV) if s["lengths"] is None else s["lengths"].long()
    there = (torch.arange(T, device=DEV) < n[:, None])[:, :, None, None]
    kk, vv = torch.where(there, k, 0), torch.where(there, v, 0)
    decay = torch.exp(g)[:, None, None]
    x = None if s0 is None else decay * s0.detach()
    out = _plain_scan(q, kk, vv, g, x, None if s0 is None else n - 1)
    end = None
    if s0 is not None:
        out, end = out
        end = torch.where((n > 0).view(B, 1, 1, 1), end, s0.detach())
    o = torch.where(there, out * scale, 0).to(q.dtype)
    if s["kind"] == "memory":
        return o if end is None else (o, end)
    go = torch.where(there, s["go"], 0).float() * scale
    dq = torch.where(there, _plain_scan(go, vv, kk, g, None if x is None else x.transpose(-1, -2)), 0).to(q.dtype)
    # backwards in time: R_j = e^g R_(j + 1) + scale q_j go_j^T
    rq, rk, rv, rgo = (_flip(t, n) for t in (torch.where(there, q, 0).float(), kk.float(), vv.float(), go))
    gs = s["gs"]
    dk_ = _flip(_plain_scan(rv, rgo, rq, g, None if gs is None else gs.transpose(-1, -2)), n)
    dv_ = _plain_scan(rk, rq, rgo, g, gs, None if s0 is None else n - 1)
    ds = ()
    if s0 is not None:
        dv_, first = dv_
        ds = (torch.where((n > 0).view(B, 1, 1, 1), decay * first, gs),)
    grads = (dq, dk_.to(k.dtype), _flip(dv_, n).to(v.dtype), *ds)
    return (o, *grads) if end is None else (o, end, *grads)


def _plain_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    s["next"].copy_(torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., None] * v[..., None, :])
    o = s["scale"] * (q[..., None] * s["next"]).sum(2)
    return o.to(s["q"].dtype), s["next"]


def run(s):
    kind = s["kind"]
    if not own:
        with torch.no_grad():
            return _plain_norm(s) if kind.startswith("norm") else _plain_step(s) if kind == "step" else _plain_memory(s)
    from codecoder_b200 import ops
    if kind.startswith("norm"):
        y = ops.group_norm(s["x"], s["groups"], s["w"], s["b"], EPS, s["act"], DTYPES[s["y"]])
        if kind == "norm":
            return y
        return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["gy"]))
    if kind == "step":
        return ops.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["scale"],
                                         new_state=s["next"]), s["next"]
    out = ops.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["s0"], s["lengths"],
                               return_state=s["s0"] is not None)
    if kind == "memory":
        return out
    if s["s0"] is None:
        return (out.detach(), *torch.autograd.grad(out, s["leaves"], s["go"]))
    return (out[0].detach(), out[1].detach(), *torch.autograd.grad(out, s["leaves"], (s["go"], s["gs"])))


def work(case):
    e = SIZE[case["x"]]
    if case["kind"].startswith("norm"):
        C, y = case["channels"], SIZE[case["y"]]
        n = case["samples"] * case["rows"] * C
        affine = 8 * C if case["affine"] else 0
        if case["kind"] == "norm":
            return dict(bytes=n * (e + y) + affine, flops=8 * n)
        return dict(bytes=2 * n * (e + y) + 2 * affine, flops=24 * n)       # x, gy in; y, dx out
    B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    state = 4 * B * H * dk * dv
    if case["kind"] == "step":
        return dict(bytes=2 * state + B * H * (2 * dk + 2 * dv) * e + 4 * H, flops=5 * B * H * dk * dv)
    T = case["length"]
    tokens = B * T * H * (0.5 if case["ragged"] else 1.0)                   # lengths are spread evenly over 0 .. T
    outs = B * T * H                                                        # written whole
    # a token's products: with the state, or with the tokens before it
    per = min(4 * dk * dv, (dk + dv) * (T + 1))
    ends = 2 * state if case["state"] else 0                                # the state in and out
    if case["kind"] == "memory":
        return dict(bytes=tokens * (2 * dk + dv) * e + outs * dv * e + ends, flops=tokens * per)
    return dict(bytes=tokens * (2 * dk + 2 * dv) * e + outs * (2 * dk + 2 * dv) * e + 2 * ends, flops=tokens * 4 * per)


def _exact_norm(case, s):
    B, N, C, G = case["samples"], case["rows"], case["channels"], case["groups"]
    train = case["kind"] == "norm train"
    x = s["x"].detach().double().requires_grad_(train)
    w = b = None
    if case["affine"]:
        w, b = (s[n].detach().double().requires_grad_(train) for n in "wb")
    var, mean = torch.var_mean(x.view(B, N, G, -1), dim=(1, 3), correction=0, keepdim=True)
    z = ((x.view(B, N, G, -1) - mean) * torch.rsqrt(var + EPS)).view(B, N, C)
    if w is not None:
        z = torch.addcmul(b, z, w)
    if case["act"] == "silu":
        z = torch.nn.functional.silu(z)
    elif case["act"] == "gelu":
        z = torch.nn.functional.gelu(z, approximate="tanh")
    if not train:
        return z
    leaves = [x] if w is None else [x, w, b]
    return (z.detach(), *torch.autograd.grad(z, leaves, s["gy"].double()))


def _exact_memory(case, s):
    """The recurrence in blocks, one after the other, and its gradients by autograd."""
    train = case["kind"] == "memory train"
    q, k, v = (s[n].detach().double().requires_grad_(train) for n in "qkv")
    B, T, H, dk = q.shape
    s0 = s["s0"].detach().double().requires_grad_(train) if case["state"] else None
    n = torch.full((B,), T, device=DEV) if s["lengths"] is None else s["lengths"].long()
    g = s["log_decay"].double()
    S = q.new_zeros(B, H, dk, case["dv"]) if s0 is None else s0
    L, outs = 128, []
    for t0 in range(0, T, L):
        l = min(L, T - t0)
        i = torch.arange(l, device=DEV)
        have = (n - t0).clamp(0, l)                                         # this block's tokens of each sequence
        live = (i < have[:, None]).double()[:, :, None, None]
        qb, kb, vb = (t[:, t0:t0 + l] * live for t in (q, k, v))
        lag = (i[:, None] - i[None, :]).double()
        d = torch.tril(torch.exp(g[:, None, None] * lag.clamp_min(0)))
        p = torch.einsum("bihd,bjhd->bhij", qb, kb) * d
        past = torch.exp(g[:, None] * (i + 1).double())                     # (H, l)
        o = torch.einsum("bhij,bjhe->bihe", p, vb) + torch.einsum("bihd,hi,bhde->bihe", qb, past, S)
        outs.append(o * s["scale"])
        rest = torch.exp(g[None, :, None] * (have[:, None, None] - 1 - i).clamp_min(0).double())      # (B, H, l)
        S = torch.exp(g[None] * have[:, None].double())[..., None, None] * S + torch.einsum("bihd,bhi,bihe->bhde", kb, rest, vb)
    o = torch.cat(outs, 1)
    if not train:
        return o if s0 is None else (o, S)
    if s0 is None:
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), s["go"].double()))
    return (o.detach(), S.detach(), *torch.autograd.grad((o, S), (q, k, v, s0), (s["go"].double(), s["gs"].double())))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("norm"):
        return _exact_norm(case, s)
    if case["kind"] == "step":
        S = torch.exp(s["log_decay"].double())[:, None, None] * s["state"].double()
        S += torch.einsum("bhd,bhe->bhde", s["k"].double(), s["v"].double())
        return torch.einsum("bhd,bhde->bhe", s["q"].double(), S) * s["scale"], S
    return _exact_memory(case, s)
