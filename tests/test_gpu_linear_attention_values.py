"""Values that are not finite in linear attention, where the weight that they are multiplied by is zero: a decay whose powers
underflow or that forgets everything, a scale of zero.  Zero times NaN is NaN by the definition, whichever kernel runs."""
import pytest
import torch

from codecoder_b200 import ops
from test_gpu_linear_attention import BF16, F32, HALF, U, definition, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,at", [(2, 0), (5, 1), (8, 7), (9, 0), (16, 3), (16, 15), (17, 3), (40, 20)])
@pytest.mark.parametrize("where", ["q", "k", "v", "go"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_weights_of_zero_do_not_hide_them(dtype, T, at, where, value):
    for scale, D in ((1.0, (16, 16)), (1.0, (32, 24)), (0.0, (32, 32))):
        s = make(2, T, 4, *D, dtype, T + at)
        s["g"] = torch.tensor([-200.0, -float("inf"), 0.0, -90.0], device=DEV)
        s[where][1, at, :, 3] = value
        want = definition(s["q"], s["k"], s["v"], s["g"], scale, None, None, s["go"])
        leaves = [s[x].requires_grad_() for x in ("q", "k", "v")]
        o = ops.linear_attention(*leaves, s["g"], scale)
        grads = torch.autograd.grad(o, leaves, s["go"])
        for what, a, b in zip(("o", "dq", "dk", "dv"), (o, *grads), (want[0], *want[2:5])):
            lost = a.isfinite() & ~b.isfinite()
            assert not bool(lost.any()), (what, scale, int(lost.sum()))
            # the other sequence, and what has no part in it at all, are as they are
            spread = ~a.isfinite() & b.isfinite()
            assert not bool(spread[0].any()), (what, scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_sequence_shows_what_its_steps_show(dtype):
    """And may show it up to 31 positions before as well."""
    T = 16
    s = make(1, T, 2, 32, 32, dtype, 5)
    s["g"] = torch.tensor([-150.0, -float("inf")], device=DEV)
    s["v"][0, 4, :, 7] = float("nan")
    o = ops.linear_attention(s["q"], s["k"], s["v"], s["g"])
    state = torch.zeros(1, 2, 32, 32, device=DEV)
    for t in range(T):
        z = ops.linear_attention_step(s["q"][:, t], s["k"][:, t], s["v"][:, t], s["g"], state)
        assert not bool((z.isnan() & ~o[:, t].isnan()).any()) and bool(z[..., 7].isnan().all()) == (t >= 4), t


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 7, 8, 9, 16, 17])
def test_a_scale_of_zero_and_decays_that_underflow(dtype, T):
    """Finite values stay as they were: zeros with a scale of zero, a row's own product where the decay leaves nothing else.  A sum
    of D products of D, each (D + 48) 2^-24 of its magnitudes at most (128 more of bf16 parts), rounded once."""
    s = make(2, T, 3, 32, 32, dtype, T)
    s["g"] = torch.tensor([-200.0, -float("inf"), -0.5], device=DEV)
    leaves = [s[x].requires_grad_() for x in ("q", "k", "v")]
    o = ops.linear_attention(*leaves, s["g"], 0.0)
    for t in (o, *torch.autograd.grad(o, leaves, s["go"])):
        assert bool((t == 0).all())
    o = ops.linear_attention(*leaves, s["g"], 1.0)
    grads = torch.autograd.grad(o, leaves, s["go"])
    args = (s["q"].detach(), s["k"].detach(), s["v"].detach(), s["g"], 1.0, None, None, s["go"])
    want, mag = definition(*args), definition(*args, mag=True)
    for a, i in zip((o, *grads), (0, 2, 3, 4)):
        e = (32 + 4 * T + 48 + (128 if dtype == BF16 else 0)) * U * mag[i]
        assert bool(((a.detach().double() - want[i]).abs() <= e + (want[i].abs() + e) * HALF[dtype] + 1e-36).all())
