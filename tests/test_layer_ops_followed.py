"""Forward-mode tangents and traces, which the kernels do not take part in, are refused and not dropped: a result without a tangent
is a derivative of zero, and a traced call's a constant.  Runs without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from codecoder_b200 import ops


@pytest.fixture(scope="module", autouse=True)
def built():
    from codecoder_b200.build import build
    build()


def calls():
    """Each differentiable input of each function in turn: (call, its arguments, the place)."""
    x, w = torch.randn(2, 3, 8), torch.ones(8)
    norm = [x, w, w.clone()]
    for i in range(3):
        yield lambda *a: ops.group_norm(a[0], 2, a[1], a[2]), norm, i
    q = torch.randn(2, 3, 2, 4)
    whole = [q, q.clone(), q.clone(), -torch.ones(2), torch.zeros(2, 2, 4, 4)]
    for i in range(5):
        yield lambda *a: ops.linear_attention(*a[:4], state=a[4]), whole, i
    step = [t[:, 0].clone() for t in whole[:3]] + whole[3:]
    for i in range(5):
        yield ops.linear_attention_step, step, i


@pytest.mark.parametrize("at", range(13))
@pytest.mark.parametrize("no_grad", [False, True])
def test_tangents_are_refused(at, no_grad):
    f, args, i = list(calls())[at]
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        dual = [fwd.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(args)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(*dual)


@pytest.mark.parametrize("at", [0, 3, 8])
def test_traces_are_refused(at):
    f, args, _ = list(calls())[at]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda *a: f(*a), tuple(args), check_trace=False)


def test_a_tangent_of_the_state_written_is_refused():
    """It would be left beside a value that it no longer belongs to."""
    q, g, state = torch.randn(2, 2, 4), -torch.ones(2), torch.zeros(2, 2, 4, 4)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        ops.linear_attention_step(q, q, q, g, state, new_state=fwd.make_dual(state.clone(), state))
