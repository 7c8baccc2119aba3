"""The embedding gradient on small whole numbers: every partial sum is a whole number below 2^24, so fp32 adds them without
rounding in any order and the results have to be equal, not near."""
import pytest
import torch

from codecoder_b200 import _lib, ops

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


def test_the_sort_by_passes_gives_the_same_bits(monkeypatch):
    """Where the sort's cluster cannot be resident the launches per pass take its place, at any size: the same order of the
    positions, so the same gradient bit for bit."""
    for n, V, C in ((1, 9, 4), (100, 300, 7), (2047, 70000, 8), (2049, 9, 64), (8192, 500, 20), (30000, 1 << 17, 4),
                    (65536, 4096, 33)):
        g = torch.Generator(device=DEV).manual_seed(n)
        ids = torch.randint(-1, V + 1, (n,), generator=g, device=DEV)
        gy = torch.randn(n, C, generator=g, device=DEV)
        monkeypatch.delenv("BPC_EMBED_SORT", raising=False)
        want = ops.embed_wgrad(gy, ids, V)
        monkeypatch.setenv("BPC_EMBED_SORT", "passes")
        assert torch.equal(ops.embed_wgrad(gy, ids, V), want)
        assert torch.equal(ops.embed_wgrad(gy, ids.int(), V), want)


def test_the_sort_by_passes_is_what_the_variable_selects(monkeypatch):
    """The launches per pass write their digit counts behind the two lists of pairs; the cluster keeps its counts on chip."""
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    n, V, C = 1000, 300, 8
    ids, gy = torch.randint(0, V, (n,), device=DEV), torch.randn(n, C, device=DEV)
    dw = torch.empty(V, C, device=DEV)
    need = int(L.bpc_embed_wgrad_workspace_size(n, V, C))
    lists = 2 * ((8 * n + 255) // 256 * 256)
    for how, counts in (("passes", True), ("", False)):
        monkeypatch.setenv("BPC_EMBED_SORT", how)
        ws = torch.full((need,), 5, device=DEV, dtype=torch.uint8)
        _lib.check(L.bpc_embed_wgrad(gy.data_ptr(), ids.data_ptr(), 8, dw.data_ptr(), ws.data_ptr(), need, n, V, C, C, 1.0,
                                     0, 0, st), "wgrad")
        assert bool((ws[lists:lists + 1024] != 5).any()) == counts
