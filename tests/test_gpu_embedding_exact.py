"""The embedding gradient on small whole numbers: every partial sum is a whole number below 2^24, so fp32 adds them without
rounding in any order and the results have to be equal, not near."""
import pytest
import torch

from codecoder_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("V", [4, 9])
def test_the_largest_number_of_positions(V):
    """2^31 - 1 rows of one channel: places are counted up to the last one and beyond it without wrapping."""
    torch.cuda.empty_cache()
    n = 2**31 - 1
    g = torch.Generator(device=DEV).manual_seed(V)
    ids = torch.randint(0, V, (n,), generator=g, device=DEV, dtype=torch.int32)
    ids[-100:] = V - 1                                          # the last rows of the last token
    gy = torch.zeros(n, 1, device=DEV, dtype=BF16)
    at = torch.randint(0, n, (5000,), generator=g, device=DEV).unique()
    gy[at, 0] = torch.randint(-3, 4, (len(at),), generator=g, device=DEV).to(BF16)
    gy[-100:] = 1
    at = torch.cat([at[at < n - 100], torch.arange(n - 100, n, device=DEV)])
    want = torch.zeros(V, 1, device=DEV, dtype=torch.float64).index_add_(0, ids[at].long(), gy[at].double())
    assert torch.equal(ops.embed_wgrad(gy, ids, V).double(), want)
    assert ops.op_status() == 0
