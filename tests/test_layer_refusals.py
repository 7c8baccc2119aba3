"""Calls of the layers and of linear attention that have no answer are refused with a reason.  Runs without a GPU."""
import pytest
import torch

from codecoder_b200.geometry import RotatedSurface
from codecoder_b200.modules import CascadeBlock, CascadeStack


@pytest.mark.parametrize("H", [64, 512])
def test_the_fused_path_refuses_blocks_with_group_norm(H):
    blocks = [CascadeBlock(H, RotatedSurface(3, 3), 2, norm=n, groups=8) for n in ("batch", "group")]
    h = torch.zeros(1, blocks[0].c2d_all.shape[0], H)
    with pytest.raises(ValueError, match="group"):
        CascadeStack.forward_blocks(blocks, h)


@pytest.mark.parametrize("device,error,text", [("cpu", RuntimeError, "CUDA"), pytest.param("cuda", ValueError, "head size", marks=pytest.mark.gpu)])
def test_heads_of_no_size_are_refused_by_the_entry_points(device, error, text):
    from codecoder_b200 import ops
    g = torch.zeros(2, device=device)
    for shape in ((2, 3, 2, 0), ()):
        q = torch.zeros(shape, device=device)
        with pytest.raises(error, match=text):
            ops.linear_attention(q, q, q, g)
    q = torch.zeros(2, 2, 0, device=device)
    with pytest.raises(error, match=text):
        ops.linear_attention_step(q, q, q, g, torch.zeros(2, 2, 0, 0, device=device))
