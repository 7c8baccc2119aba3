"""The embedding gradient on small whole numbers: every partial sum is a whole number below 2^24, so fp32 adds them without
rounding in any order and the results have to be equal, not near."""
import pytest
import torch

from codecoder_b200 import _lib, ops
from test_gpu_embedding import make_ids

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def whole(n, C, dtype, seed, ld=None):
    """(n, C) whole numbers from -3 to 3, in rows ld apart: a sum of n of them stays below 2^24 for n up to 5.5 M"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-3, 4, (n, ld or C), generator=g, device=DEV, dtype=torch.int8).to(dtype)[:, :C]


def check_exact(gy, ids, V):
    i = ids.reshape(-1).long()
    ok = (i >= 0) & (i < V)
    want = torch.zeros(V, gy.shape[-1], device=DEV, dtype=torch.float64)
    want.index_add_(0, i[ok], gy.reshape(-1, gy.shape[-1])[ok].double())     # exact too: whole numbers below 2^53
    got = ops.embed_wgrad(gy, ids, V)
    assert got.dtype == F32
    wrong = got.double() != want
    assert not bool(wrong.any()), (int(wrong.sum()), wrong.nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 3, 4, 5, 6, 8, 9, 40, 3000])
def test_long_sums(V, dtype):
    """Every form of reading the rows (whole runs, a copy per row, unaligned, single elements) over many stages and blocks,
    with tokens that reach over many workers."""
    for C, ld in ((96, 96), (96, 104), (45, 45), (64, 65), (1, 1), (33, 40)):
        for n in (300000, 100003):
            gy = whole(n, C, dtype, V + C, ld)
            for kind in ("uniform", "padded", "hot", "one", "runs"):
                check_exact(gy, make_ids(n, V, kind, V + n), V)


@pytest.mark.parametrize("V", [4, 5, 8, 30])
def test_long_sums_of_wide_rows(V):
    for C, ld, dtype in ((512, 512, F32), (512, 520, BF16), (1100, 1100, BF16), (2304, 2304, F16), (777, 777, F32)):
        gy = whole(60001, C, dtype, V + C, ld)
        for kind in ("uniform", "hot", "last"):
            check_exact(gy, make_ids(60001, V, kind, C), V)


@pytest.mark.parametrize("n", [8192, 8193, 16384, 16385, 32768, 32769, 65535, 65536, 65537, 200001])
def test_sorts_at_the_sizes_where_they_change(n):
    for V, C, dtype in ((9, 3, BF16), (255, 20, F32), (256, 20, F16), (70000, 8, BF16), (1 << 17, 4, F32), (1 << 24, 1, F16)):
        gy = whole(n, C, dtype, n + V)
        for kind in ("uniform", "padded", "hot", "runs"):
            check_exact(gy, make_ids(n, V, kind, n + V, torch.int32 if V % 2 else torch.int64), V)


def test_the_stems_of_the_networks():
    """The Cascade stem's training batch (512 shots of 504 nodes, 512 channels, fp32, int64 ids of 5 tokens) and the d = 11
    pre-decoder's rows as its unfused network has them (fp32, int64)."""
    check_exact(whole(512 * 504, 512, F32, 1).view(512, 504, 512), make_ids(512 * 504, 5, "uniform", 2).view(512, 504), 5)
    check_exact(whole(1024 * 1320, 96, F32, 3), make_ids(1024 * 1320, 4, "hot", 4), 4)


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
