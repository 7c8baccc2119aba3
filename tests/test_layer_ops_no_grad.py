"""Decays that are a parameter: refused where a gradient of theirs would be expected, taken where none is."""
import pytest
import torch

from codecoder_b200 import ops


def test_refused_only_where_a_gradient_is_expected():
    q, g = torch.zeros(2, 3, 2, 4), torch.zeros(2, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        ops.linear_attention(q, q, q, g)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode(), pytest.raises(RuntimeError, match="CUDA"):         # the tensors' device is looked at next
            ops.linear_attention(q, q, q, g)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 40])
def test_without_a_gradient_they_are_decays(T):
    q, k, v = torch.randn(3, 2, T, 3, 16, device="cuda")
    g = torch.tensor([-0.1, -1.0, -3.0], device="cuda")
    want = ops.linear_attention(q, k, v, g, return_state=True)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = ops.linear_attention(q, k, v, g.clone().requires_grad_(), return_state=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
