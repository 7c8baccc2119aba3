"""The embedding and gradient-norm entry points refuse bad arguments on the host, before any device work; empty calls
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


def test_embed_lookup_refusals(lib):
    f = lib.bpc_embed_lookup
    refused(f(16, 8, 16, 16, -1, 5, 8, 8, 1.0, F32, F32, None), "positions")
    refused(f(16, 8, 16, 16, 1 << 31, 5, 8, 8, 1.0, F32, F32, None), "positions")
    refused(f(16, 8, 16, 16, 4, 0, 8, 8, 1.0, F32, F32, None), "tokens")
    refused(f(16, 8, 16, 16, 4, 2**31 - 1, 8, 8, 1.0, F32, F32, None), "tokens")
    refused(f(16, 8, 16, 16, 4, 5, 0, 8, 1.0, F32, F32, None), "channels")
    refused(f(16, 2, 16, 16, 4, 5, 8, 8, 1.0, F32, F32, None), "int32 or int64")
    refused(f(16, 8, 16, 16, 4, 5, 8, 8, 1.0, 3, F32, None), "dtype")
    refused(f(16, 8, 16, 16, 4, 5, 8, 8, 1.0, F32, -1, None), "dtype")
    refused(f(16, 8, 16, 16, 4, 5, 8, 7, 1.0, F32, F32, None), "stride")
    refused(f(12, 8, 16, 16, 4, 5, 8, 8, 1.0, F32, F32, None), "aligned")
    refused(f(16, 8, 18, 16, 4, 5, 8, 8, 1.0, F32, F32, None), "aligned")
    refused(f(16, 8, 16, 17, 4, 5, 8, 8, 1.0, F32, BF16, None), "aligned")
    for k in range(3):
        p = [16, 16, 16]
        p[k] = None
        refused(f(p[0], 8, p[1], p[2], 4, 5, 8, 8, 1.0, F32, F32, None), "null")
    assert f(None, 8, None, None, 0, 5, 8, 8, 1.0, F32, F32, None) == 0


def test_embed_wgrad_refusals(lib):
    f = lib.bpc_embed_wgrad
    need = lib.bpc_embed_wgrad_workspace_size(100, 5, 8)
    assert need > 0
    big = 1 << 40
    refused(f(16, 16, 8, 16, 16, big, -1, 5, 8, 8, 1.0, F32, F32, None), "positions")
    refused(f(16, 16, 8, 16, 16, big, 100, 0, 8, 8, 1.0, F32, F32, None), "tokens")
    refused(f(16, 16, 16, 16, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "int32 or int64")
    refused(f(16, 16, 8, 16, 16, big, 100, 5, 8, 8, 1.0, F32, 7, None), "dtype")
    refused(f(16, 16, 8, 16, 16, big, 100, 5, 8, 4, 1.0, F32, F32, None), "stride")
    refused(f(16, 16, 8, None, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "null dw")
    refused(f(16, 16, 8, 18, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "aligned")
    refused(f(18, 16, 8, 16, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "aligned")
    refused(f(16, 16, 8, 16, 8, big, 100, 5, 8, 8, 1.0, F32, F32, None), "workspace")
    refused(f(None, 16, 8, 16, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "null")
    refused(f(16, None, 8, 16, 16, big, 100, 5, 8, 8, 1.0, F32, F32, None), "null")
    refused(f(16, 16, 8, 16, None, big, 100, 5, 8, 8, 1.0, F32, F32, None), "null")
    refused(f(16, 16, 8, 16, 16, need - 1, 100, 5, 8, 8, 1.0, F32, F32, None), "workspace", code=6)
    assert lib.bpc_embed_wgrad_workspace_size(0, 5, 8) == 0
    assert lib.bpc_embed_wgrad_workspace_size(10, 0, 8) == 0


def lists(*entries):
    """(address, count, dtype) entries as the host arrays of a list"""
    return (array("Q", [e[0] for e in entries]), array("q", [e[1] for e in entries]), array("i", [e[2] for e in entries]))


def at(a):
    return a.buffer_info()[0]


def clip(lib, ins, outs, max_norm=1.0, norm=16, ws=16, ws_bytes=1 << 40):
    p, n, d = lists(*ins)
    q, _, e = lists(*outs)
    return lib.bpc_clip_grads(at(p), at(q), at(n), at(d), at(e), len(ins), max_norm, norm, ws, ws_bytes, None)


def test_grad_norm_refusals(lib):
    def f(entries, norm=16, ws=16, ws_bytes=1 << 40):
        p, n, d = lists(*entries)
        return lib.bpc_grad_norm(at(p), at(n), at(d), len(entries), norm, ws, ws_bytes, None)
    ok = (4096, 10, F32)
    refused(f([ok], norm=None), "null")
    refused(f([ok], ws=None), "null")
    refused(f([ok], norm=18), "aligned")
    refused(f([ok], ws=12), "aligned")
    refused(f([ok], ws_bytes=lib.bpc_grad_norm_workspace_size(1) - 1), "workspace", code=6)
    refused(f([(4096, -1, F32)]), "element count")
    refused(f([(4096, 2**62, F32)]), "element count")
    refused(f([(4096, 2**42, F32)]), "too many")
    refused(f([(4096, 10, 5)]), "dtype")
    refused(f([ok, (0, 10, F32)]), "null tensor")
    refused(f([ok, (4098, 10, F32)]), "aligned")
    refused(lib.bpc_grad_norm(None, None, None, 1, 16, 16, 1 << 40, None), "null")
    refused(lib.bpc_grad_norm(None, None, None, -1, 16, 16, 1 << 40, None), "tensors")
    assert lib.bpc_grad_norm_workspace_size(-1) == 0
    assert lib.bpc_grad_norm_workspace_size(5000) > lib.bpc_grad_norm_workspace_size(1000) >= 8


def test_clip_grads_refusals(lib):
    a, b = (4096, 10, F32), (8192, 10, F32)
    for bad in (-1.0, float("nan")):
        refused(clip(lib, [a], [a], max_norm=bad), "max_norm")
    refused(clip(lib, [a], [(0, 10, F32)]), "null tensor")
    refused(clip(lib, [a], [(8192, 10, 4)]), "dtype")
    refused(clip(lib, [a], [(8193, 10, BF16)]), "aligned")
    # the same gradient twice, an output on another input or output, a shifted copy of its own input
    refused(clip(lib, [a, a], [a, a]), "overlaps")
    refused(clip(lib, [a, b], [b, (16384, 10, F32)]), "overlaps")
    refused(clip(lib, [a, b], [(16384, 10, F32), (16384 + 36, 10, F32)]), "overlaps")
    refused(clip(lib, [b, a], [b, (8192 - 36, 10, F32)]), "overlaps")
    refused(clip(lib, [a], [(4100, 10, F32)]), "overlaps")
    # in place means the same type too
    refused(clip(lib, [a], [(4096, 10, BF16)]), "overlaps")
    refused(lib.bpc_clip_grads(4096, None, 4096, 4096, 4096, 1, 1.0, None, 16, 1 << 40, None), "null")


def test_python_refusals():
    ids, w = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embed_lookup(ids, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embedding(ids, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embed_wgrad(torch.zeros(3, 8), ids, 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.grad_norm([w])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.clip_grads([w], 1.0)
    with pytest.raises(ValueError, match="at least one"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="at least one"):
        ops.clip_grads(iter([]), 1.0)
    assert float(ops.clip_grad_norm_([torch.nn.Parameter(w)], 1.0)) == 0.0      # no gradients: nothing to do
