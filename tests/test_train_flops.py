"""The training step's algorithmic FLOPs count the memory's maps and its attention.  Runs without a GPU."""
from dataclasses import replace

import pytest
import torch
import torch.nn.functional as F
from torch.utils.flop_counter import FlopCounterMode

from codecoder_b200.geometry import RotatedSurface
from codecoder_b200.params import CONFIGS
from codecoder_b200.train import train_flops_per_shot


@pytest.mark.parametrize("d,heads", [(3, 1), (5, 3), (7, 4)])
def test_a_memory_is_counted(d, heads):
    cfg = replace(CONFIGS["d11_train"], d=d, rounds=d, layers=2)
    g, C = RotatedSurface(d, d), cfg.channels
    if C % heads:
        heads = 2
    more = train_flops_per_shot(g, cfg, heads) - train_flops_per_shot(g, cfg)
    # the maps by torch's own count, forward and backward
    x = torch.zeros(g.N_d, C, requires_grad=True)
    w = [torch.zeros(C, C, requires_grad=True) for _ in range(4)]
    with FlopCounterMode(display=False) as counted:
        sum(F.linear(x, p).sum() for p in w).backward()
    # the attention pair by pair: every position with those up to its own, a product and a weighted sum of D each, in each of
    # four scans; or through the state, an update and a product of D x D
    D = C // heads
    pairs = sum(2 * 2 * D * (t + 1) for t in range(g.R)) * (g.N_d // g.R) * heads
    assert more == counted.get_total_flops() + 4 * min(pairs, 4 * D * D * g.N_d * heads)


def test_without_a_memory_the_count_is_as_it_was():
    cfg = CONFIGS["d11_train"]
    g = RotatedSurface(cfg.d, cfg.rounds)
    assert train_flops_per_shot(g, cfg) == train_flops_per_shot(g, cfg, None) == \
        6.0 * cfg.K * cfg.channels**2 * (cfg.layers * g.N_d + (cfg.layers - 1) * g.N_c) + 12.0 * cfg.channels * g.N_d
