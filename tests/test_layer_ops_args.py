"""The group-norm and linear-attention entry points refuse bad arguments on the host, before any device work; empty calls
are no-ops.  Runs without a GPU."""
from array import array

import pytest
import torch

from codecoder_b200 import _lib, ops

F32, BF16, F16 = _lib.BPC_DTYPE_F32, _lib.BPC_DTYPE_BF16, _lib.BPC_DTYPE_F16


@pytest.fixture(scope="module")
def lib():
    from codecoder_b200.build import build
    build()
    return _lib.lib()


def refused(rc, text, code=2):
    assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())


def call(f, args, **changes):
    return f(*{**args, **changes}.values())


def test_group_norm_refusals(lib):
    f = lib.bpc_group_norm_fwd
    ok = dict(x=16, y=16, stats=None, w=None, b=None, B=2, N=3, C=8, G=2, ss=24, rs=8, eps=1e-5, act=1, xt=F32,
              yt=BF16, ws=16, wsb=1 << 40, st=None)
    for name in ("x", "y", "ws"):
        refused(call(f, ok, **{name: None}), "null")
    refused(call(f, ok, B=-1), "samples")
    refused(call(f, ok, N=-1), "samples")
    refused(call(f, ok, B=1 << 30, N=1 << 30), "samples")
    refused(call(f, ok, C=0), "channels")
    refused(call(f, ok, C=1 << 21), "channels")
    refused(call(f, ok, G=3), "divide")
    refused(call(f, ok, G=0), "divide")
    refused(call(f, ok, act=3), "activation")
    refused(call(f, ok, xt=7), "dtype")
    refused(call(f, ok, xt=BF16, yt=F32), "dtype")
    refused(call(f, ok, rs=-8), "strides")
    refused(call(f, ok, eps=-1e-5), "eps")
    refused(call(f, ok, eps=float("nan")), "eps")
    for name, at in (("x", 18), ("y", 17), ("stats", 20), ("w", 18), ("b", 18), ("ws", 8)):
        refused(call(f, ok, **{name: at}), "aligned")
    refused(call(f, ok, wsb=0), "workspace", code=6)
    assert call(f, ok, B=0, x=None, y=None) == 0 and call(f, ok, N=0, x=None, y=None) == 0
    size = lib.bpc_group_norm_workspace_size
    assert size(0, 3, 8, 2, F32, 0) == 0 and size(2, 3, 8, 3, F32, 0) == 0 and size(2, 3, 8, 2, 9, 0) == 0


def test_group_norm_backward_refusals(lib):
    f = lib.bpc_group_norm_bwd
    ok = dict(gy=16, x=16, stats=16, w=None, b=None, dx=16, dw=16, db=16, B=2, N=3, C=8, G=2, gs=24, gr=8, xs=24, xr=8,
              act=1, xt=F32, yt=BF16, ws=16, wsb=1 << 40, st=None)
    for name in ("gy", "x", "stats", "ws"):
        refused(call(f, ok, **{name: None}), "null")
    refused(call(f, ok, G=5), "divide")
    refused(call(f, ok, gr=-1), "strides")
    refused(call(f, ok, act=-1), "activation")
    refused(call(f, ok, xt=F16, yt=BF16), "dtype")
    for name, at in (("gy", 17), ("x", 18), ("dx", 18), ("stats", 20), ("w", 18), ("b", 18), ("dw", 18), ("db", 18),
                     ("ws", 8)):
        refused(call(f, ok, **{name: at}), "aligned")
    refused(call(f, ok, wsb=0), "workspace", code=6)
    assert call(f, ok, B=0, dw=None, db=None, gy=None, x=None) == 0


def strides(*s):
    a = array("q", s)
    return a, a.buffer_info()[0]


def test_linear_attention_refusals(lib):
    f = lib.bpc_linear_attention_fwd
    keep, st = strides(*(24, 8, 4) * 3)
    ok = dict(q=16, k=16, v=16, o=16, g=16, s=None, ns=None, n=None, nb=0, B=2, T=3, H=2, dk=4, dv=4, strides=st, scale=1.0,
              dt=F32, ws=16, wsb=1 << 40, stream=None)
    for name in ("q", "k", "v", "o", "g", "ws", "strides"):
        refused(call(f, ok, **{name: None}), "null")
    for name in ("B", "T", "H"):
        refused(call(f, ok, **{name: -1}), "negative")
    refused(call(f, ok, B=1 << 20, H=1 << 10), "2^30")
    refused(call(f, ok, T=(1 << 30) + 1), "2^30")
    for name in ("dk", "dv"):
        for d in (0, 129):
            refused(call(f, ok, **{name: d}), "head sizes")
    refused(call(f, ok, dt=F16), "dtype")
    refused(call(f, ok, scale=float("inf")), "scale")
    refused(call(f, ok, n=16, nb=2), "lengths")
    refused(call(f, ok, n=20, nb=8), "lengths")
    for name, at in (("q", 18), ("k", 18), ("v", 18), ("o", 18), ("ws", 8)):
        refused(call(f, ok, **{name: at}), "aligned")
    refused(call(f, ok, s=20), "aligned")
    refused(call(f, ok, ns=24), "aligned")
    keep2, bad = strides(*(24, 8, 4) * 2, 24, -8, 4)
    refused(call(f, ok, strides=bad), "strides")
    refused(call(f, ok, wsb=0), "workspace", code=6)
    assert call(f, ok, B=0) == 0 and call(f, ok, H=0) == 0 and call(f, ok, T=0) == 0
    assert lib.bpc_linear_attention_workspace_size(2, 3, 2, 4, 129, F32, 0) == 0


def test_linear_attention_backward_refusals(lib):
    f = lib.bpc_linear_attention_bwd
    keep, st = strides(*(24, 8, 4) * 4)
    ok = dict(q=16, k=16, v=16, go=16, g=16, s=None, gs=None, fw=None, n=None, nb=0, dq=16, dk_=16, dv_=16, ds=None, B=2, T=3, H=2, dk=4,
              dv=4, strides=st, scale=1.0, dt=F32, ws=16, wsb=1 << 40, stream=None)
    for name in ("q", "k", "v", "go", "g", "dq", "dk_", "dv_", "ws", "strides"):
        refused(call(f, ok, **{name: None}), "null")
    for name in ("q", "k", "v", "go", "dq", "dk_", "dv_"):
        refused(call(f, ok, **{name: 18}), "aligned")
    for name in ("s", "gs", "ds", "fw"):
        refused(call(f, ok, **{name: 24}), "aligned")
    refused(call(f, ok, dk=200), "head sizes")
    refused(call(f, ok, wsb=0), "workspace", code=6)
    assert call(f, ok, B=0) == 0 and call(f, ok, T=0) == 0


def test_linear_attention_step_refusals(lib):
    f = lib.bpc_linear_attention_step
    keep, st = strides(*(8, 4) * 3)
    ok = dict(q=16, k=16, v=16, o=16, g=16, s=4096, ns=4096, B=2, H=2, dk=4, dv=4, strides=st, scale=1.0, dt=BF16, stream=None)
    for name in ("q", "k", "v", "o", "g", "s", "ns", "strides"):
        refused(call(f, ok, **{name: None}), "null")
    for name in ("q", "k", "v", "o"):
        refused(call(f, ok, **{name: 17}), "aligned")
    refused(call(f, ok, s=4098), "aligned")
    # 256 bytes of state: one buffer, or two apart
    refused(call(f, ok, ns=4096 + 240), "overlaps")
    refused(call(f, ok, ns=4096 - 240), "overlaps")
    refused(call(f, ok, dv=129), "head sizes")
    assert call(f, ok, B=0) == 0


def test_python_refusals():
    x, q = torch.zeros(2, 3, 8), torch.zeros(2, 3, 2, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm(x.requires_grad_(), 2)
    with pytest.raises(ValueError, match="activation"):
        ops.group_norm(x, 2, activation="tanh")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(2, 2, 4, 4))
    with pytest.raises(ValueError, match="gradient"):
        ops.linear_attention(q, q, q, torch.zeros(2, requires_grad=True))


def test_layers_cast_and_prepared():
    from codecoder_b200.geometry import RotatedSurface
    from codecoder_b200.modules import CascadeBlock, RoundMemory
    m = RoundMemory(32, 2, 5)
    rates = m.log_decay.clone()
    assert m.bfloat16().log_decay.dtype == torch.float32 and torch.equal(m.log_decay, rates)
    assert m.q.dtype == torch.bfloat16 and m.double().q.dtype == torch.float64 and torch.equal(m.log_decay, rates)
    kept = m.log_decay
    assert m.to("cpu").log_decay is kept
    blk = CascadeBlock(64, RotatedSurface(3, 3), 1, norm="group", groups=8)
    assert blk.prepare_inference() is blk
