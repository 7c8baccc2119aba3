"""The layers on the group-norm and linear-attention operators, and the networks that take them, against the same
compositions in 64 bits.

Tolerances: relative to max |ref|; 1e-4 for fp32 networks and 5e-2 for gradients under bf16 autocast, as the networks' other
tests (every stored activation and gradient is rounded to bf16 along the way).  A layer alone in fp32, and the operators as
they are used together: 1e-4 behind the norm, 1e-5 for states.  The norm divides a head's result by its own deviation, which
in a first round is |q k| and may be nearly nothing: plain fp32 arithmetic is off by up to 1.3e-5 in the gradients of these
layers, and 3e-7 of o's root mean square (a third of 2^-24 sqrt(T + D) times the products of a product, the operator's usual
error in fp32), put into the 64-bit composition as noise, makes 1.4e-5 of the results and 5.3e-5 of the gradients."""
import os
from dataclasses import replace

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from codecoder_b200.geometry import RotatedSurface
from codecoder_b200.modules import CascadeBlock, CascadeNet, CascadeStack, GroupNorm, RoundMemory
from codecoder_b200.params import CONFIGS, init_params
from codecoder_b200.sampler import sample, sample_torch
from codecoder_b200.train import PreDecoderNet, Trainer
from oracle import predecoder_oracle as orc
from test_cascade_net import net_geo
from test_gpu_cascade import bb72_geo
from test_gpu_linear_attention import definition

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).abs().max() / b.abs().max().clamp_min(1e-30))


class Norm64(torch.nn.Module):
    """GroupNorm by torch, in the type of its input."""

    def __init__(self, gn):
        super().__init__()
        self.groups, self.eps = gn.groups, gn.eps
        self.weight, self.bias = (torch.nn.Parameter(t.detach().double().cpu()) for t in (gn.weight, gn.bias))

    def forward(self, x):
        C = x.shape[-1]
        y = F.group_norm(x.reshape(x.shape[0], -1, C).transpose(1, 2), self.groups, self.weight, self.bias, self.eps)
        return F.silu(y.transpose(1, 2).reshape(x.shape))


class Memory64(torch.nn.Module):
    """RoundMemory in 64 bits: the recurrence round by round, with autograd's gradients."""

    def __init__(self, m):
        super().__init__()
        self.C, self.heads, self.D = m.C, m.heads, m.D
        for n in ("q", "k", "v", "out"):
            setattr(self, n, torch.nn.Parameter(getattr(m, n).detach().double().cpu()))
        self.norm = Norm64(m.norm)
        self.decay = torch.exp(m.log_decay.double().cpu())[:, None, None]

    def forward(self, x):
        B, T, S, C = x.shape
        q, k, v = (F.linear(x, w).view(B, T, S * self.heads, self.D) for w in (self.q, self.k, self.v))
        state, outs = 0.0, []
        for t in range(T):
            state = self.decay * state + k[:, t, :, :, None] * v[:, t, :, None, :]
            outs.append((q[:, t, :, None] @ state)[:, :, 0] * self.D**-0.5)
        o = torch.stack(outs, 1).view(B * T * S, C)
        return x + F.linear(self.norm(o), self.out).view(x.shape)


def make_memory(C, heads, sites, seed):
    m = RoundMemory(C, heads, sites, seed).to(DEV)
    g = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        m.out.copy_(torch.randn(C, C, generator=g) / C**0.5)
        m.norm.weight.copy_(1 + 0.2 * torch.randn(C, generator=g))
        m.norm.bias.copy_(0.2 * torch.randn(C, generator=g))
    return m


@pytest.mark.parametrize("C,heads,S,T", [(96, 3, 9, 11), (64, 2, 25, 40), (20, 5, 4, 3)])
def test_round_memory_matches_the_recurrence(C, heads, S, T):
    m = make_memory(C, heads, S, T)
    ref = Memory64(m)
    x = torch.randn(3, T, S, C, generator=torch.Generator().manual_seed(T))
    gy = torch.randn(3, T, S, C, generator=torch.Generator().manual_seed(T + 1))
    xd, xr = x.to(DEV).requires_grad_(), x.double().requires_grad_()
    y, yr = m(xd), ref(xr)
    assert rel(y, yr) < 1e-4
    y.backward(gy.to(DEV))
    yr.backward(gy.double())
    assert rel(xd.grad, xr.grad) < 1e-4
    for n, p in m.named_parameters():
        assert rel(p.grad, dict(ref.named_parameters())[n].grad) < 1e-4, n
    # a whole experiment, or its rounds one by one
    state = m.start(3)
    for t in range(T):
        z = m.step(xd.detach()[:, t], state)
        assert rel(z, y[:, t]) < 1e-4
    _, end = m(xd.detach(), return_state=True)
    assert rel(state, end) < 1e-5
    # or in two parts, with what the first leaves behind
    if T > 5:
        a, mid = m(xd.detach()[:, :5], return_state=True)
        b = m(xd.detach()[:, 5:], state=mid)
        assert rel(torch.cat([a, b], 1), y) < 1e-4


def test_round_memory_of_experiments_of_different_lengths():
    """A shot among others and by itself: products of other shapes, whose sums are rounded in another order.  q, k and v
    (about 0.6) are sums of 32 products, sqrt(32) 2^-24 0.6 = 2e-7 apart, so o = sum of 16 q S / 4 is about
    sqrt(16) / 4 3 2e-7 0.6^2 = 2e-7 apart.  The norm divides that by sqrt(var + eps), in a first round whose q is nearly
    orthogonal to its k by no more than sqrt(eps) = 1 / 316: 6e-5, and the map back (16 such values, weights 1 / sqrt(32))
    makes 4.5e-5 of it, or 1.3e-5 of max |y| = 3.5.  fp32 arithmetic on the CPU in two orders: up to 7e-6 in 60 draws."""
    m = make_memory(32, 2, 5, 3)
    x = torch.randn(4, 12, 5, 32, device=DEV)
    n = torch.tensor([12, 0, 5, 1], device=DEV)
    y, state = m(x, lengths=n, return_state=True)
    for b, k in enumerate(n.tolist()):
        assert torch.equal(y[b, k:], x[b, k:])          # nothing there: passed through
        if k:
            z, s = m(x[b:b + 1, :k], return_state=True)
            assert rel(y[b, :k], z[0]) < 2e-5 and rel(state[b], s[0]) < 1e-6
    assert bool((state[1] == 0).all())


def test_a_memory_in_bf16_keeps_its_rates():
    """The layer cast to bf16 is its own operators on its bf16 weights with the rates in fp32, bit for bit.  (Against the fp32
    layer no tolerance holds: the norm divides by what is left of q k, whose rounding is relative to |q| |k|.)"""
    from codecoder_b200 import ops
    m = make_memory(64, 2, 9, 5)
    x = torch.randn(2, 20, 9, 64, device=DEV)
    rates = m.log_decay.clone()
    m.bfloat16()
    assert torch.equal(m.log_decay, rates) and m.log_decay.device == rates.device
    xb = x.bfloat16()
    y, state = m(xb, return_state=True)
    q, k, v = (F.linear(xb, w).view(2, 20, 18, 32) for w in (m.q, m.k, m.v))
    o, want = ops.linear_attention(q, k, v, rates, return_state=True)
    n = ops.group_norm(o.view(-1, 64), 2, m.norm.weight, m.norm.bias, activation="silu")
    assert y.dtype == torch.bfloat16 and torch.equal(y, xb + F.linear(n, m.out).view(x.shape)) and torch.equal(state, want)
    steps = m.start(2)
    for t in range(20):
        m.step(x[:, t].bfloat16(), steps)
    # k and v of products of other shapes: a rounding apart in places, 2^-7 of a term; the terms' sum is a few times the largest
    assert rel(steps, state) < 10 * 2**-8
    with pytest.raises(TypeError, match="fp32 or bf16"):
        m.half()(x.half())


def test_a_new_memory_is_the_identity():
    m = RoundMemory(64, 2, 9).to(DEV)
    x = torch.randn(2, 3, 9, 64, device=DEV)
    assert torch.equal(m(x), x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(m(x.bfloat16()), x.bfloat16())


def nets(cfg, seed, memory, **kw):
    g = RotatedSurface(cfg.d, cfg.rounds)
    params = init_params(cfg, seed)
    net = PreDecoderNet(g, cfg, params, memory=memory, seed=seed).to(DEV)
    net.memory = make_memory(cfg.channels, memory, g.n_data_round, seed)
    ref = PreDecoderNet(g, cfg, params, gmm=lambda x, w, idx, inv: orc.gather_mm(x, w, idx.cpu())).double()
    ref.memory = Memory64(net.memory)
    return g, net, ref


@pytest.mark.parametrize("autocast", [False, True])
def test_predecoder_net_with_a_memory_matches_64_bits(autocast):
    cfg = replace(CONFIGS["d11_train"], d=5, rounds=5, layers=2) if autocast else replace(CONFIGS["d5_fp32"], d=3, rounds=3, layers=2)
    g, net, ref = nets(cfg, 41, 3 if autocast else 1)
    det, err = sample(g, 0.03, 40, 42)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        z = net(torch.as_tensor(det).to(DEV))
        loss = net(torch.as_tensor(det).to(DEV), torch.as_tensor(err).to(DEV))
    loss.backward()
    zr = ref(torch.as_tensor(det))
    F.binary_cross_entropy_with_logits(zr, torch.as_tensor(err).double()).backward()
    assert rel(z, zr) < (3e-2 if autocast else 1e-4)
    pr = dict(ref.named_parameters())
    for n, p in net.named_parameters():
        if p.requires_grad:
            assert rel(p.grad, pr[n].grad) < (5e-2 if autocast else 1e-4), (n, rel(p.grad, pr[n].grad))


def test_a_new_memory_leaves_the_network_as_it_was():
    cfg = replace(CONFIGS["d11_train"], d=5, rounds=5, layers=2)
    g = RotatedSurface(cfg.d, cfg.rounds)
    det, err = sample_torch(g, 0.03, 64, 3, device=DEV)
    out = []
    for memory in (None, 3):
        net = PreDecoderNet(g, cfg, init_params(cfg, 4), memory=memory).to(DEV)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out.append((net(det).detach(), net(det, err).detach()))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_graphed_training_steps_with_a_memory_match_eager_steps():
    cfg = replace(CONFIGS["d11_train"], d=5, rounds=5, layers=2)
    g = RotatedSurface(cfg.d, cfg.rounds)
    batches = [sample_torch(g, 0.03, 128, 70 + i, device=DEV) for i in range(3)]
    make = lambda: Trainer(PreDecoderNet(g, cfg, init_params(cfg, 59), memory=3).to(DEV), lr=1e-3, graph=True)
    eager, graphed = make(), make()
    le = [eager.step(*batches[0]) for _ in range(2)] + [eager.step(*batches[i]) for i in (0, 1, 2)]
    lg = [graphed.step_graphed(*batches[i]) for i in (0, 1, 2)]
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(le[2:]), torch.stack(lg))
    for (n, a), b in zip(eager.model.named_parameters(), graphed.model.parameters()):
        assert torch.equal(a, b), n
    assert float(eager.model.memory.out.detach().abs().max()) > 0           # the memory has begun to take part


def group_block(golden_dir, H, res):
    conv_z = dict(np.load(os.path.join(golden_dir, "bb72_c14_conv.npz")))
    torch.manual_seed(6)
    blk = CascadeBlock(H, bb72_geo(conv_z), 4, res=res, norm="group", groups=8)
    with torch.no_grad():
        for p in blk.parameters():
            p.add_(0.1 * torch.randn(p.shape) * p.abs().mean())
    return blk.to(DEV)


def block64(blk):
    """The block's composition in 64 bits on the CPU, sharing nothing but its tables."""
    import copy
    ref = copy.deepcopy(blk).double().cpu()
    for n in ("gn1", "gn2", "gn3"):
        setattr(ref, n, Norm64(getattr(blk, n)))
    conv = ref.conv

    def forward(x):
        data = torch.cat([orc.gather_mm(x, conv.w_c2d[d], getattr(conv, f"c2d{d}")) for d in range(len(conv.w_c2d))], 1)
        return torch.cat([orc.gather_mm(data, conv.w_d2c[c], getattr(conv, f"d2c{c}")) for c in range(len(conv.w_d2c))], 1)
    conv.forward = forward
    return ref


@pytest.mark.parametrize("res", ["branch", "skip"])
def test_cascade_block_with_group_norm_matches_64_bits(golden_dir, res):
    blk = group_block(golden_dir, 64, res)
    ref = block64(blk)
    N = blk.c2d_all.shape[0]
    h = torch.randn(2, 504, 64, generator=torch.Generator().manual_seed(2))
    hd, hr = h.to(DEV).requires_grad_(), h.double().requires_grad_()
    y, yr = blk(hd), ref(hr)
    assert N == 504 and rel(y, yr) < 1e-4
    gy = torch.randn(h.shape, generator=torch.Generator().manual_seed(3))
    y.backward(gy.to(DEV))
    yr.backward(gy.double())
    assert rel(hd.grad, hr.grad) < 1e-4
    pr = dict(ref.named_parameters())
    for n, p in blk.named_parameters():
        assert rel(p.grad, pr[n].grad) < 1e-4, n
    # eval is the same composition, and a shot's result is its own
    with torch.no_grad():
        assert torch.equal(blk.eval()(hd), blk.train()(hd))
        assert rel(blk(hd[1:]), y[1:]) < 1e-5
        assert torch.equal(CascadeStack([blk]).eval()(hd), blk(hd))


def test_cascade_net_with_group_norm_trains(golden_dir):
    z = dict(np.load(os.path.join(golden_dir, "cascade_net_bb72.npz")))
    conv_z = dict(np.load(os.path.join(golden_dir, "bb72_c14_conv.npz")))
    torch.manual_seed(8)
    net = CascadeNet(net_geo(z, conv_z), int(z["H"]), 2, z["det_t"], z["det_typ"], z["det_site"], z["logicals"],
                     res=str(z["res"]), norm="group").to(DEV)
    assert not any("bn" in n for n in net.state_dict()) and "gn_out.weight" in net.state_dict()
    det = torch.as_tensor(z["det"]).to(DEV)
    ref = net.train()(det)
    with torch.no_grad():
        assert torch.equal(net.eval()(det), net(det)) and rel(net(det), ref) < 1e-5
    net.train()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = net(det)
    assert rel(y, ref) < 5e-2
    y.float().square().sum().backward()
    ref.square().sum().backward()
    for n, p in net.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), n


def test_a_run_of_the_operators_as_they_are_used_together():
    """Projection, attention over the rounds, head-wise norm, and back, against the definitions in 64 bits."""
    from codecoder_b200 import ops
    B, T, H, D = 4, 23, 6, 32
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(B, T, H, D, generator=g, device=DEV).requires_grad_() for _ in range(3))
    w = (1 + 0.1 * torch.randn(H * D, generator=g, device=DEV)).requires_grad_()
    decay = torch.log1p(-torch.exp2(-torch.linspace(1, 6, H, device=DEV)))
    o, state = ops.linear_attention(q, k, v, decay, return_state=True)
    y = ops.group_norm(o.reshape(B * T, H * D), H, w, activation="silu")
    gy = torch.randn(y.shape, generator=g, device=DEV)
    grads = torch.autograd.grad(y, (q, k, v, w), gy)
    o64, s64 = definition(q.detach(), k.detach(), v.detach(), decay, D**-0.5, None, None)
    leaf = o64.clone().requires_grad_()
    w64 = w.detach().double().requires_grad_()
    x = leaf.view(B * T, H, D)
    var, mean = torch.var_mean(x, dim=2, correction=0, keepdim=True)
    y64 = F.silu(((x - mean) / (var + 1e-5).sqrt()).reshape(B * T, H * D) * w64)
    go, gw = torch.autograd.grad(y64, (leaf, w64), gy.double())
    want = definition(q.detach(), k.detach(), v.detach(), decay, D**-0.5, None, None, go)
    assert rel(y, y64) < 1e-4 and rel(state, s64) < 1e-5 and rel(grads[3], gw) < 1e-4
    for a, b in zip(grads, want[2:5]):
        assert rel(a, b) < 1e-4
    # the next round goes on from there
    nxt = [torch.randn(B, H, D, generator=g, device=DEV) for _ in range(3)]
    o1 = ops.linear_attention_step(*nxt, decay, state.detach())
    whole = [torch.cat([a.detach(), b[:, None]], 1) for a, b in zip((q, k, v), nxt)]
    assert rel(o1, definition(*whole, decay, D**-0.5, None, None)[0][:, -1]) < 1e-5


def test_refusals():
    with pytest.raises(ValueError, match="groups"):
        GroupNorm(48, 32)
    with pytest.raises(ValueError, match="heads"):
        RoundMemory(96, 5, 4)
    with pytest.raises(ValueError, match="heads"):
        RoundMemory(512, 2, 4)
    with pytest.raises(ValueError, match="norm"):
        CascadeBlock(64, RotatedSurface(3), 1, norm="layer")
