"""The embedding and clipping operators where the networks and the trainer call them, and at the sizes where their kernels
change form.  Tolerances: a token's sum of m rows in fp32 is off by at most (m + 1) 2^-24 sum |x|, and its rounding; see
test_gpu_embedding.py."""
import os
import subprocess
import sys
from dataclasses import replace

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from codecoder_b200 import _lib, ops
from codecoder_b200.geometry import RotatedSurface
from codecoder_b200.params import CONFIGS, init_params
from codecoder_b200.sampler import sample_torch
from codecoder_b200.train import PreDecoderNet, Trainer
from test_cascade_net import make_net
from test_gpu_embedding import BF16, F16, F32, check_lookup, check_wgrad, make_ids

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_cascade_net_trains_on_the_embedding_op(golden_dir):
    """The stem through ops.embedding: the same values as nn.functional.embedding, and a gradient that is the sum of the
    stream's gradient by token."""
    z = dict(np.load(os.path.join(golden_dir, "cascade_net_bb72.npz")))
    conv_z = dict(np.load(os.path.join(golden_dir, "bb72_c14_conv.npz")))
    net = make_net(z, conv_z).to(DEV).train()
    seen = {}

    def lookup(tok, weight):
        h = ops.embedding(tok, weight)
        assert torch.equal(h, F.embedding(tok, weight))
        h.register_hook(lambda g: seen.update(tok=tok, g=g.detach().clone()))
        return h

    net.embedding = lookup
    det = torch.as_tensor(z["det"]).to(DEV)
    net(det).square().sum().backward()
    check_wgrad(net.embed.weight.grad, seen["g"], seen["tok"], 5, 1.0, F32)
    # the same network, the default lookup: the same output
    net.embedding = None
    a = net(det)
    net.embedding = ops.embedding
    assert torch.equal(a, net(det))


def test_unfused_predecoder_net_takes_the_embedding_op():
    cfg = replace(CONFIGS["d5_fp32"], d=3, rounds=3, layers=2)
    g = RotatedSurface(cfg.d, cfg.rounds)
    det, err = sample_torch(g, 0.05, 32, 7, device=DEV)
    out = []
    for embedding in (F.embedding, ops.embedding):
        net = PreDecoderNet(g, cfg, init_params(cfg, 5), embedding=embedding).to(DEV)
        loss = net(det, err)
        loss.backward()
        out.append((loss.detach(), net.embed.grad))
    assert torch.equal(out[0][0], out[1][0])
    # two fp32 sums of the same at most 32 x 24 rows
    assert float((out[0][1] - out[1][1]).abs().max()) <= 2 * 769 * 2.0**-24 * 768 * float(out[0][1].abs().max())


def test_unfused_predecoder_nets_embedding_gradient_is_its_streams_sum():
    """The table's gradient against the sum by token of the stream's own gradient: at most 768 rows of one token."""
    cfg = replace(CONFIGS["d5_fp32"], d=3, rounds=3, layers=2)
    g = RotatedSurface(cfg.d, cfg.rounds)
    det, err = sample_torch(g, 0.05, 32, 7, device=DEV)
    seen = {}

    def lookup(tok, weight):
        h = ops.embedding(tok, weight)
        h.register_hook(lambda gh: seen.update(tok=tok, g=gh.detach().clone()))
        return h

    net = PreDecoderNet(g, cfg, init_params(cfg, 5), embedding=lookup).to(DEV)
    net(det, err).backward()
    check_wgrad(net.embed.grad, seen["g"], seen["tok"], net.embed.shape[0], 1.0, F32)


def test_trainer_clips_with_the_library():
    """Trainer(clip_grad=ops.clip_grad_norm_): eager and graphed steps give the same bits, and one step's update is that
    of torch's clipping to rounding (Adam's first step is lr times the gradient's sign where it is not tiny)."""
    cfg = replace(CONFIGS["d11_train"], d=5, rounds=5, layers=3)
    g = RotatedSurface(cfg.d, cfg.rounds)
    batches = [sample_torch(g, 0.03, 256, 60 + i, device=DEV) for i in range(3)]
    make = lambda **kw: Trainer(PreDecoderNet(g, cfg, init_params(cfg, 59)).to(DEV), lr=1e-3, clip=1e-3, graph=True, **kw)
    eager, graphed = (make(clip_grad=ops.clip_grad_norm_) for _ in range(2))
    le = [eager.step(*batches[0]) for _ in range(2)] + [eager.step(*batches[i]) for i in (0, 1, 2)]
    lg = [graphed.step_graphed(*batches[i]) for i in (0, 1, 2)]
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(le[2:]), torch.stack(lg))
    for a, b in zip(eager.model.parameters(), graphed.model.parameters()):
        assert torch.equal(a, b)
    norms = []
    for f in (torch.nn.utils.clip_grad_norm_, ops.clip_grad_norm_):
        t = make(clip_grad=lambda ps, m, f=f: norms.append((f(ps, m), [p.grad.clone() for p in ps])))
        t.step(*batches[1])
    (n0, g0), (n1, g1) = norms
    assert abs(float(n0) - float(n1)) <= 1e-5 * float(n0) and float(n0) > 1e-3
    for a, b in zip(g0, g1):
        assert bool(((a - b).abs() <= 1e-5 * a.abs() + 1e-30).all())


@pytest.mark.parametrize("n", [8192, 8193, 16384, 16385, 32768, 32769, 65535, 65536, 65537, 200001])
def test_sorts_at_the_sizes_where_they_change(n):
    for V, C, kind in ((9, 3, "uniform"), (300, 20, "hot"), (70000, 8, "padded"), (1 << 17, 4, "runs")):
        gy = torch.randn(n, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)).to(BF16)
        ids = make_ids(n, V, kind, n + V, torch.int32 if V == 300 else torch.int64)
        check_wgrad(ops.embed_wgrad(gy, ids, V), gy, ids, V, 1.0, F32)


@pytest.mark.parametrize("C", [1, 2, 5, 31, 33, 64, 128, 129, 250, 256, 384, 512, 514, 640, 1000, 1024, 1536, 2050, 5000])
@pytest.mark.parametrize("gt,dt", [(F32, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
def test_channel_counts_of_every_form(C, gt, dt):
    for n, V, kind in ((700, 5, "padded"), (700, 8, "uniform"), (901, 90, "hot"), (130, 400, "padded")):
        gy = (torch.randn(n, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(C + n)) / 8).to(gt)
        ids = make_ids(n, V, kind, n + C)
        check_wgrad(ops.embed_wgrad(gy, ids, V, 0.5, dt), gy, ids, V, 0.5, dt)
        w = torch.randn(V, C, device=DEV).to(gt)
        check_lookup(ops.embed_lookup(ids, w, 2.0, dt), ids, w, 2.0, dt)


@pytest.mark.parametrize("V", [1, 4, 5, 6, 8, 9, 40])
def test_rows_at_strides_and_offsets(V):
    """gy as a slice of wider rows, from every element offset, 16- and 32-bit; dW and W inside larger buffers at theirs."""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    n = 3000
    ids = make_ids(n, V, "padded", V)
    for gt, code in ((F32, 0), (BF16, 1)):
        for C, ld, off in ((64, 64, 0), (64, 72, 8), (64, 65, 1), (64, 64, 2), (96, 200, 4), (45, 45, 0), (45, 45, 3), (45, 64, 0),
                           (256, 256, 1), (1024, 1024, 0), (1024, 1032, 8), (2304, 2304, 0)):
            buf = torch.randn(n * ld + 64, device=DEV).to(gt)
            gy = buf[off:off + n * ld].view(n, ld)[:, :C]
            for woff in (0, 1, 2, 4):
                dbuf = torch.full((V * C + 64,), 7.0, device=DEV)
                dw = dbuf[woff:woff + V * C]
                need = int(L.bpc_embed_wgrad_workspace_size(n, V, C))
                ws = torch.empty(need, device=DEV, dtype=torch.uint8)
                _lib.check(L.bpc_embed_wgrad(gy.data_ptr(), ids.data_ptr(), 8, dw.data_ptr(), ws.data_ptr(), need, n, V, C,
                                             ld, 1.0, code, 0, st), "wgrad")
                check_wgrad(dw.view(V, C), gy, ids, V, 1.0, F32)
                assert bool((dbuf[:woff] == 7).all()) and bool((dbuf[woff + V * C:] == 7).all())
    assert ops.op_status() == 0


def test_few_tokens_over_many_stages_and_far_rows():
    """Enough rows for every block to go round its ring several times, and rows whose offsets pass 32 bits."""
    for C, V, gt in ((96, 4, BF16), (96, 5, F32), (7, 3, F16), (512, 8, BF16)):
        n = 400000 if C < 512 else 120000
        gy = torch.randn(n, C, device=DEV).to(gt)
        ids = make_ids(n, V, "padded", C)
        dw = ops.embed_wgrad(gy, ids, V)
        check_wgrad(dw, gy, ids, V, 1.0, F32)
        assert torch.equal(dw, ops.embed_wgrad(gy, ids, V))
    n, C = 5, 64
    buf = torch.zeros((n - 1) * (1 << 29) + C, device=DEV, dtype=BF16)      # rows 1 GB apart
    gy = buf.as_strided((n, C), (1 << 29, 1))
    gy.copy_(torch.randn(n, C))
    for V in (3, 30):
        ids = torch.tensor([0, 2, 2, 0, 1], device=DEV)
        check_wgrad(ops.embed_wgrad(gy, ids, V), gy, ids, V, 1.0, F32)
    w = gy                                                                    # and a table whose rows are that far apart
    assert torch.equal(ops.embed_lookup(torch.tensor([4, 0, 3, 9], device=DEV)[:3], w), w[[4, 0, 3]])
    assert ops.op_status() == 0


def test_outputs_and_inputs_past_32_bits():
    """More than 2^32 elements on either side: the last rows are as right as the first."""
    g = torch.Generator(device=DEV).manual_seed(3)
    w = torch.randn(7, 4001, device=DEV, generator=g).to(BF16)               # an odd width, and a wide one
    for table in (w, w[:, :4000].contiguous()):
        ids = torch.randint(-1, 8, (1100000,), device=DEV, generator=g)
        y = ops.embed_lookup(ids, table)
        assert y.numel() > 2**32
        for part in (slice(0, 300), slice(-300, None), slice(1073000, 1074000)):
            check_lookup(y[part], ids[part], table, 1.0, BF16)
        del y
    V, C, n = 1100000, 4000, 400                                              # 17.6 GB of gradient, nearly all zeros
    ids = torch.randint(0, V, (n,), device=DEV, generator=g)
    ids[0], ids[1] = V - 1, 0
    gy = torch.randn(n, C, device=DEV, generator=g)
    dw = ops.embed_wgrad(gy, ids, V)
    used = ids.unique()
    check_wgrad(dw[used], gy, torch.searchsorted(used, ids), len(used), 1.0, F32)
    assert int(torch.count_nonzero(dw.view(torch.int32).view(-1)[:2**31])) + \
        int(torch.count_nonzero(dw.view(torch.int32).view(-1)[2**31:])) <= len(used) * C
    del dw
    n, C = 47000000, 96                                                       # 4.5 G values: counts of ones are exact
    gy = torch.ones(n, C, device=DEV, dtype=BF16)
    ids = torch.randint(0, 4, (n,), device=DEV, generator=g, dtype=torch.int32)
    for V, t in ((4, ids), (40, ids * 11)):
        dw = ops.embed_wgrad(gy, t, V)
        want = torch.bincount(t, minlength=V).double()[:, None]
        assert bool(((dw.double() - want).abs() <= want * 2.0**-23).all())
    assert ops.op_status() == 0
    x = torch.ones(2**32 + 77, device=DEV, dtype=F16)                         # one tensor of more than 2^32 elements
    assert abs(float(ops.grad_norm([x, x[:5]])) - (2**32 + 82) ** 0.5) <= 65537 * 2.0**-24
    ops.clip_grads([x], 32768.0)
    assert bool((x[-100:] == 0.5).all()) and bool((x[:100] == 0.5).all()) and bool((x[2**31 - 50:2**31 + 50] == 0.5).all())


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing: each has the workspace it was called with."""
    n = 60000
    work = []
    for k, (V, C) in enumerate(((5, 128), (900, 128), (5, 96), (3000, 64))):
        gy = torch.randn(n, C, device=DEV).to(BF16)
        ids = make_ids(n, V, "hot", k)
        work.append((gy, ids, V, ops.embed_wgrad(gy, ids, V)))
    lists = [[torch.randn(50000 + k, device=DEV) for k in range(5)] for _ in range(2)]
    norms = [ops.grad_norm(ts) for ts in lists]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for rep in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                for gy, ids, V, want in work[k::2]:
                    got.append((ops.embed_wgrad(gy, ids, V), want))
                got.append((ops.grad_norm(lists[k]), norms[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


def test_first_calls_inside_a_capture():
    """A process whose very first calls are captured: nothing they set up on the host is refused by the capture."""
    code = """
import torch
from codecoder_b200 import ops
ids = torch.randint(0, 5, (4000,), device="cuda"); big = torch.randint(0, 900, (4000,), device="cuda")
gy = torch.randn(4000, 64, device="cuda"); w = torch.randn(5, 64, device="cuda"); outs = [torch.empty_like(gy), torch.empty_like(w)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.embed_lookup(ids, w); a = ops.embed_wgrad(gy, ids, 5); b = ops.embed_wgrad(gy, big, 900)
    n = ops.clip_grads([gy, w], 1.0, out=outs)
g.replay(); torch.cuda.synchronize()
assert torch.equal(y, w[ids]) and torch.equal(a, ops.embed_wgrad(gy, ids, 5)) and torch.equal(b, ops.embed_wgrad(gy, big, 900))
assert torch.equal(n, ops.grad_norm([gy, w]))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_captured_forward_backward_and_clipping():
    """A training step's forward, backward and in-place clipping replayed with new gradients and ids.  (No eager graph of
    the table is alive at the capture: torch's gradient accumulator would tie it to the eager stream.)"""
    w = torch.nn.Parameter(torch.randn(50, 64, device=DEV))
    ids, gy = torch.randint(0, 50, (800,), device=DEV), torch.randn(800, 64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.embedding(ids, w), w, gy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dw, = torch.autograd.grad(ops.embedding(ids, w), w, gy)
        norm = ops.clip_grads([dw], 0.5)
    for seed in (1, 2):
        ids.copy_(make_ids(800, 50, "padded", seed))
        gy.normal_()
        g.replay()
        want = ops.embed_wgrad(gy, ids, 50)
        check_wgrad(want, gy, ids, 50, 1.0, F32)
        assert torch.equal(norm, ops.clip_grads([want], 0.5)) and torch.equal(dw, want)
