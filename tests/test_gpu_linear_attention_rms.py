"""fp32 linear attention against a loss of bits: the root mean square of its errors, u = 2^-24.  An operand in two tf32 parts loses
its last bit where the second part has 12 (every fourth time on average: 0.7 u of it), and the product of the second parts,
(2^-11 / sqrt 3)^2, is left out: 0.6 u, so a product is off by sqrt(2 0.7^2 + 0.6^2) = 1.2 u, and a result has two in a row.  Each of
the 3 D / 8 steps of a sum on the tensor unit cuts off about 0.6 u: 2 u for D = 32, 3 for 64, twice.  The weights' powers are
off by up to 4 u alike for all of a chunk, and by as much again for each chunk of 32 positions that a state passes, of which
decays as these leave few.  Together about (6 + T / 32) u for independent errors, of which three times as much is allowed.
(Measured: 3.4 u for D = 16, 5 to 6 for 32, 11 for 64 and 20 for 128; what the unit cuts off is not independent, and adds up with D.)"""
import pytest
import torch

from codecoder_b200 import ops
from test_gpu_linear_attention import F32, U, definition, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,dk,dv", [(64, 5, 25, 32, 32), (32, 8, 8, 16, 16), (64, 11, 9, 32, 32), (16, 16, 8, 32, 32), (8, 40, 8, 64, 64),
                                         (4, 100, 6, 128, 128), (9, 333, 5, 24, 40), (2, 1500, 3, 64, 64)])
@pytest.mark.parametrize("with_state", [False, True])
def test_fp32_errors_are_a_few_roundings(B, T, H, dk, dv, with_state):
    s = make(B, T, H, dk, dv, F32, T + dk, with_state)
    want = definition(s["q"], s["k"], s["v"], s["g"], dk**-0.5, s["s0"], None, s["go"], s["gs"])
    leaves = [s[x].requires_grad_() for x in ("q", "k", "v", "s0") if s[x] is not None]
    out = ops.linear_attention(*leaves[:3], s["g"], state=leaves[3] if with_state else None, return_state=with_state)
    outs, gouts = (list(out), [s["go"], s["gs"]]) if with_state else ([out], [s["go"]])
    got = [*outs, *torch.autograd.grad(outs, leaves, gouts)]
    refs = [want[0], *want[1:2], *want[2:6]] if with_state else [want[0], *want[2:5]]
    rms = {}
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dstate") if with_state else ("o", "dq", "dk", "dv"), got, refs):
        rms[name] = float(((a.detach().double() - b).square().mean() / b.square().mean()).sqrt()) / U
    print(T, dk, {k: round(v, 1) for k, v in rms.items()})
    assert max(rms.values()) <= 3 * (6 + T / 32), rms
