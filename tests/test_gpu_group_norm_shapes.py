"""Group normalisation and its gradients where the kernels' shared memory ends: fp32 samples of 257 to 512 values a group in 13 to
17 groups, whose backward pass stages 544 bytes a thread.  Tolerances as in test_gpu_group_norm.py."""
import pytest
import torch

from codecoder_b200.geometry import RotatedSurface
from codecoder_b200.modules import CascadeBlock
from test_gpu_group_norm import BF16, F32, run
from test_gpu_layers import block64, rel

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("y_dtype", [F32, BF16])
@pytest.mark.parametrize("G", [13, 14, 15, 16, 17])
@pytest.mark.parametrize("N,cg", [(1, 512), (1, 260), (5, 64), (8, 64), (33, 8), (48, 8), (64, 8), (4, 128)])
def test_fp32_samples_of_many_groups(N, cg, G, y_dtype):
    for B in (1, 7, 700):
        run(B, N, G * cg, G, "silu", F32, y_dtype, True, N + G)


def test_a_block_of_16_groups_trains_in_fp32():
    torch.manual_seed(3)
    geo = RotatedSurface(5, 2)
    blk = CascadeBlock(128, geo, 2, norm="group", groups=16).to(DEV)
    ref = block64(blk)
    h = torch.randn(3, geo.N_c, 128, generator=torch.Generator().manual_seed(4))
    gy = torch.randn(h.shape, generator=torch.Generator().manual_seed(5))
    hd, hr = h.to(DEV).requires_grad_(), h.double().requires_grad_()
    y, yr = blk(hd), ref(hr)
    y.backward(gy.to(DEV))
    yr.backward(gy.double())
    # as the networks' other fp32 tests: 1e-4 of the largest
    assert rel(y, yr) < 1e-4 and rel(hd.grad, hr.grad) < 1e-4
    pr = dict(ref.named_parameters())
    for n, p in blk.named_parameters():
        assert rel(p.grad, pr[n].grad) < 1e-4, n
