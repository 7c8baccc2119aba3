"""Measured cases of the token-embedding and gradient-clipping operators of codecoder_b200.ops.

  lookup  y[i, :] = scale W[ids[i], :], a zero row where ids[i] is outside [0, V)        ops.embed_lookup
  wgrad   dW[v, :] = scale sum over i with ids[i] = v of gy[i, :]                         ops.embed_wgrad
  train   the autograd lookup forward and backward, its weight gradient clipped in place  ops.embedding, ops.clip_grads
  norm    the 2-norm over every element of a list of gradients                            ops.grad_norm
  clip    out = g min(1, max_norm / (norm + 1e-6)) over the list, and the norm            ops.clip_grads

`run` computes a case in its plain torch form, or, where `own` is true, by the library's calls; `exact` gives the
same outputs in 64 bits from the definitions."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
#: shots x check nodes x channels of the d = 11 training step: no drawn case sums more rows
LARGEST_ROWS = 8192 * 1320
LARGEST_VALUES = LARGEST_ROWS * 96


def listed():
    return [
        # one BB72 shot (504 nodes, 5 detector tokens) through a 512-channel stem: latency
        dict(name="lookup one shot", kind="lookup", rows=504, tokens=5, channels=512, weight="f32", out="f32",
             scale=1.0, ids="syndrome", pad=0.0, ids32=False),
        # the stem of a Cascade network's training batch: 512 BB72 shots
        dict(name="lookup batch", kind="lookup", rows=512 * 504, tokens=5, channels=512, weight="f32", out="f32",
             scale=1.0, ids="syndrome", pad=0.0, ids32=False),
        # a large vocabulary of odd size, bf16, scaled by sqrt(channels), some positions padded
        dict(name="lookup vocabulary", kind="lookup", rows=32768, tokens=50021, channels=1024, weight="bf16",
             out="bf16", scale=32.0, ids="zipf", pad=0.05, ids32=False),
        # the weight gradient of one shot's stem: latency
        dict(name="wgrad one shot", kind="wgrad", rows=504, tokens=5, channels=512, weight="f32", out="f32",
             scale=1.0, ids="syndrome", pad=0.0, ids32=False),
        # the d = 11 training step's 8,192 shots x 1,320 checks: few tokens, millions of rows each
        dict(name="wgrad d11 batch", kind="wgrad", rows=8192 * 1320, tokens=4, channels=96, weight="f32", out="bf16",
             scale=1.0, ids="syndrome", pad=0.0, ids32=True),
        # a large vocabulary: most tokens have no row, the frequent ones thousands
        dict(name="wgrad vocabulary", kind="wgrad", rows=32768, tokens=50021, channels=1024, weight="f32", out="bf16",
             scale=32.0, ids="zipf", pad=0.05, ids32=False),
        # odd everything: a channel count that no vector width divides
        dict(name="wgrad odd", kind="wgrad", rows=4099, tokens=777, channels=45, weight="f16", out="f16",
             scale=0.5, ids="uniform", pad=0.2, ids32=True),
        # forward, backward and clipping of one embedding as a training step runs them
        dict(name="train", kind="train", rows=65536, tokens=4096, channels=512, weight="f32", out="bf16",
             scale=1.0, ids="zipf", pad=0.0, ids32=False, max_norm=1.0),
        # the gradients of the d = 11 network (19 tensors, 1.2 M values), views of one bucket as DDP keeps them
        dict(name="clip d11 network", kind="clip", tensors="predecoder", width=96, depth=6, grad="f32", out="f32",
             bucket=True, norm=4.0, max_norm=1.0),
        # the gradients of a 14-block Cascade network (176 tensors, 20 M values)
        dict(name="clip cascade network", kind="clip", tensors="cascade", width=512, depth=14, grad="f32", out="f32",
             bucket=False, norm=3.0, max_norm=1.0),
        # many small ragged tensors in bf16, below the limit's reach: the norm alone
        dict(name="norm ragged", kind="norm", tensors="ragged", width=20000, depth=300, grad="bf16", out="bf16",
             bucket=True, norm=0.5, max_norm=1.0),
        # larger than any cache: bf16 gradients clipped into fp32 ones
        dict(name="clip large", kind="clip", tensors="ragged", width=16000001, depth=40, grad="bf16", out="f32",
             bucket=False, norm=10.0, max_norm=1.0),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lookup", "lookup", "wgrad", "wgrad", "train", "norm", "clip", "clip"])
    if kind in ("lookup", "wgrad", "train"):
        tokens = rng.choice([_spread(rng, 2, 64), _spread(rng, 65, 60000)])
        channels = rng.choice([_spread(rng, 8, 2048), 8 * _spread(rng, 1, 256)])
        rows = _spread(rng, 1, min(2000000, LARGEST_VALUES // (2 * channels)))
        weight = rng.choice(["f32", "f32", "bf16", "f16"])
        out = rng.choice(["f32", "bf16"]) if weight == "f32" else weight
        case = dict(kind=kind, rows=rows, tokens=tokens, channels=channels, weight=weight, out=out,
                    scale=rng.choice([1.0, 0.5, 32.0]), ids=rng.choice(["uniform", "zipf"]),
                    pad=rng.choice([0.0, 0.1]), ids32=rng.random() < 0.5)
        if kind == "train":
            case["max_norm"] = 1.0
        return case
    tensors = rng.choice(["predecoder", "cascade", "ragged"])
    if tensors == "ragged":
        width, depth = _spread(rng, 10, 2000000), _spread(rng, 1, 400)
        depth = max(1, min(depth, 100000000 // width))
    elif tensors == "predecoder":
        width, depth = rng.choice([32, 64, 96, 128]), rng.randint(2, 12)
    else:
        width, depth = 512, rng.randint(1, 14)
    grad = rng.choice(["f32", "bf16", "f16"])
    return dict(kind=kind, tensors=tensors, width=width, depth=depth, grad=grad, out=rng.choice([grad, "f32"]),
                bucket=rng.random() < 0.5, norm=rng.choice([0.5, 4.0, 40.0]), max_norm=1.0)


def _numels(case):
    """The element counts of a gradient list."""
    w, d = case["width"], case["depth"]
    if case["tensors"] == "predecoder":      # embedding, d check -> data and 2 (d - 1) data -> check matrices, head
        return [4 * w] + (d + 2 * (d - 1)) * [8 * w * w] + [2 * w, 2]
    if case["tensors"] == "cascade":         # embedding, d bottleneck blocks, bn_out, scatter and the read-out's MLP
        b = w // 4
        block = [w, w, b, b, b, b, b * w] + 4 * [b * 12 * b] + [b * w]
        return [5 * w] + d * block + [w, w, w * 24 * w, 2 * w * w, 2 * w, 2 * w, 1]
    r = np.random.default_rng(w * 1000 + d)  # ragged: 1 .. w elements
    return [int(v) for v in r.integers(1, w + 1, d)]


def _probabilities(case):
    """The chance of each token, in the order in which they are drawn (before the vocabulary is shuffled)."""
    V = case["tokens"]
    if case["ids"] == "zipf":
        return np.diff(np.log(np.arange(1, V + 2))) / math.log(V + 1)
    if case["ids"] == "uniform":
        return np.full(V, 1.0 / V)
    p = np.array([0.475, 0.025, 0.475, 0.025])          # 2 type + bit, 5 % of the detectors set
    return p if V == 4 else np.append(p * 360 / 504, 144 / 504)      # the fifth: a node without a detector


def _ids(case, g):
    n, V = case["rows"], case["tokens"]
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    if case["ids"] == "zipf":
        t = (torch.exp(u * math.log(V + 1)) - 1).long().clamp(0, V - 1)
        t = torch.randperm(V, generator=g, device=DEV)[t]
    elif case["ids"] == "uniform":
        t = (u * V).long().clamp(0, V - 1)
    else:
        edges = torch.as_tensor(np.cumsum(_probabilities(case))[:-1], device=DEV)
        t = torch.bucketize(u, edges, right=True)
    if case["pad"]:
        t = torch.where(torch.rand(n, generator=g, device=DEV) < case["pad"], torch.full_like(t, -1), t)
    return t.int() if case["ids32"] else t


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case)
    if case["kind"] in ("lookup", "wgrad", "train"):
        s["ids"] = _ids(case, g)
        if case["kind"] != "wgrad":
            s["w"] = torch.randn(case["tokens"], case["channels"], generator=g, device=DEV).to(DTYPES[case["weight"]])
            s["w"].requires_grad_(case["kind"] == "train")
        if case["kind"] != "lookup":
            gy = torch.empty(case["rows"], case["channels"], device=DEV, dtype=DTYPES[case["out"]])
            s["gy"] = gy.normal_(0.0, 0.03125, generator=g)      # small, as a mean loss gives: fp16 sums stay finite
    else:
        numels = _numels(case)
        sigma = case["norm"] / math.sqrt(sum(numels))
        dt, out = DTYPES[case["grad"]], DTYPES[case["out"]]
        flat = torch.empty(sum(numels), device=DEV, dtype=dt).normal_(0.0, sigma, generator=g)
        s["grads"] = list(flat.split(numels))                       # views of one bucket, wherever they fall
        if not case["bucket"]:
            s["grads"] = [t.clone() for t in s["grads"]]            # tensors of their own
        if case["kind"] == "clip":
            s["flat_out"] = torch.empty(sum(numels), device=DEV, dtype=out)
            s["outs"] = list(s["flat_out"].split(numels))
    return s


def _plain_lookup(ids, w, scale, dtype):
    ok = (ids >= 0) & (ids < w.shape[0])
    y = w[ids.long().clamp(0, w.shape[0] - 1)].float() * (scale * ok[:, None])
    return y.to(dtype)


def _plain_wgrad(gy, ids, V, scale, dtype):
    # a token's sum can run over millions of rows: 64 bits for long lists
    acc = torch.float64 if ids.numel() > 65536 else torch.float32
    ok = (ids >= 0) & (ids < V)
    dw = torch.zeros(V, gy.shape[1], device=gy.device, dtype=acc)
    dw.index_add_(0, ids.long().clamp(0, V - 1), gy.to(acc) * ok[:, None])
    return (dw * scale).to(dtype)


def _plain_norm(x):
    return x.square().sum().sqrt()


def run(s):
    kind = s["kind"]
    if own:
        from codecoder_b200 import ops
        if kind == "lookup":
            return ops.embed_lookup(s["ids"], s["w"], s["scale"], DTYPES[s["out"]])
        if kind == "wgrad":
            return ops.embed_wgrad(s["gy"], s["ids"], s["tokens"], s["scale"], DTYPES[s["weight"]])
        if kind == "train":
            y = ops.embedding(s["ids"], s["w"], s["scale"], DTYPES[s["out"]])
            dw, = torch.autograd.grad(y, s["w"], s["gy"])
            norm = ops.clip_grads([dw], s["max_norm"])
            return y.detach(), dw, norm
        if kind == "norm":
            return ops.grad_norm(s["grads"])
        norm = ops.clip_grads(s["grads"], s["max_norm"], out=s["outs"])
        return s["flat_out"], norm
    if kind == "lookup":
        return _plain_lookup(s["ids"], s["w"], s["scale"], DTYPES[s["out"]])
    if kind == "wgrad":
        return _plain_wgrad(s["gy"], s["ids"], s["tokens"], s["scale"], DTYPES[s["weight"]])
    if kind == "train":
        w = s["w"].detach()
        y = _plain_lookup(s["ids"], w, s["scale"], DTYPES[s["out"]])
        dw = _plain_wgrad(s["gy"], s["ids"], s["tokens"], s["scale"], w.dtype)
        x = dw.float()
        norm = _plain_norm(x)
        return y, (x * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)).to(w.dtype), norm
    x = torch.cat([g.reshape(-1) for g in s["grads"]]).float()
    norm = _plain_norm(x)
    if kind == "norm":
        return norm
    s["flat_out"].copy_(x * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0))
    return s["flat_out"], norm


def work(case):
    if case["kind"] in ("lookup", "wgrad", "train"):
        n, V, C = case["rows"], case["tokens"], case["channels"]
        valid = n * (1.0 - case["pad"])
        ids = n * (4 if case["ids32"] else 8)
        used = float(-np.expm1(valid * np.log1p(-_probabilities(case) * (1 - 1e-12))).sum())   # tokens that occur
        ws, os_ = SIZE[case["weight"]], SIZE[case["out"]]
        lookup = dict(bytes=ids + used * C * ws + n * C * os_, flops=n * C)
        wgrad = dict(bytes=ids + valid * C * os_ + V * C * ws, flops=valid * C + V * C)
        if case["kind"] == "lookup":
            return lookup
        if case["kind"] == "wgrad":
            return wgrad
        # the ids are one input; the gradient is written once
        return dict(bytes=lookup["bytes"] + wgrad["bytes"] - ids, flops=lookup["flops"] + wgrad["flops"] + 3 * V * C)
    N = sum(_numels(case))
    if case["kind"] == "norm":
        return dict(bytes=N * SIZE[case["grad"]] + 4, flops=2 * N)
    return dict(bytes=N * (SIZE[case["grad"]] + SIZE[case["out"]]) + 4, flops=3 * N)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("lookup", "wgrad", "train"):
        V, C, n = case["tokens"], case["channels"], case["rows"]
        ids = s["ids"].long()
        ids = torch.where((ids < 0) | (ids >= V), torch.full_like(ids, V), ids)      # row V: no token
        y = dw = None
        if case["kind"] != "wgrad":
            table = torch.cat([s["w"].detach().double(), torch.zeros(1, C, device=DEV, dtype=torch.float64)])
            y = table.index_select(0, ids) * case["scale"]
        if case["kind"] != "lookup":
            # runs of the sorted ids as differences of a running sum, a block of channels at a time
            order = torch.argsort(ids, stable=True)
            ends = torch.searchsorted(ids[order], torch.arange(V, device=DEV), right=True)
            dw = torch.empty(V, C, device=DEV, dtype=torch.float64)
            step = max(1, min(C, 100000000 // max(1, n)))
            for c in range(0, C, step):
                run_ = torch.zeros(n + 1, min(step, C - c), device=DEV, dtype=torch.float64)
                torch.cumsum(s["gy"][:, c:c + step].index_select(0, order).double(), 0, out=run_[1:])
                at = run_[ends]
                dw[:, c:c + step] = torch.diff(at, dim=0, prepend=torch.zeros_like(at[:1])) * case["scale"]
        if case["kind"] == "lookup":
            return y
        if case["kind"] == "wgrad":
            return dw
        norm = torch.linalg.vector_norm(dw)
        return y, dw * min(1.0, case["max_norm"] / (float(norm) + 1e-6)), norm
    x = torch.cat([t.double().flatten() for t in s["grads"]])
    norm = torch.linalg.vector_norm(x)
    if case["kind"] == "norm":
        return norm
    return x * min(1.0, case["max_norm"] / (float(norm) + 1e-6)), norm
