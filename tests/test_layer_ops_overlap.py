"""States that share memory are refused on the host by linear attention's forward and backward entry points: one block writes a
sequence's last state while another reads its first.  Only a step updates a state in place.  Runs without a GPU."""
from array import array

import pytest

from codecoder_b200 import _lib

B, H, DK, DV = 2, 2, 4, 4
BYTES = B * H * DK * DV * 4


@pytest.fixture(scope="module")
def lib():
    from codecoder_b200.build import build
    build()
    return _lib.lib()


def forward(lib, state, new_state, T):
    s = array("q", (24, 8, 4) * 3)
    return lib.bpc_linear_attention_fwd(16, 16, 16, 16, 16, state, new_state, None, 0, B, T, H, DK, DV, s.buffer_info()[0], 1.0,
                                        _lib.BPC_DTYPE_F32, 16, 1 << 40, None)


def backward(lib, state, grad_state, dstate, T):
    s = array("q", (24, 8, 4) * 4)
    return lib.bpc_linear_attention_bwd(16, 16, 16, 16, 16, state, grad_state, None, None, 0, 16, 16, 16, dstate, B, T, H, DK, DV,
                                        s.buffer_info()[0], 1.0, _lib.BPC_DTYPE_F32, 16, 1 << 40, None)


@pytest.mark.parametrize("T", [0, 3, 1000])
@pytest.mark.parametrize("by", [0, 16, -16, BYTES - 16, 16 - BYTES])
def test_overlapping_states_are_refused(lib, T, by):
    at = 1 << 20
    assert forward(lib, at, at + by, T) == 2 and "new_state overlaps state" in _lib.last_error()
    assert backward(lib, None, at, at + by, T) == 2 and "dstate overlaps" in _lib.last_error()
    assert backward(lib, at, None, at + by, T) == 2 and "dstate overlaps" in _lib.last_error()
