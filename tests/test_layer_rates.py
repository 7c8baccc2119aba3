"""RoundMemory's decays over casts and moves of the layer: the rates that it has, the user's own too, in fp32.  Without a GPU."""
import copy

import torch

from codecoder_b200.modules import RoundMemory


def test_a_cast_keeps_the_users_rates():
    m = RoundMemory(32, 2, 5)
    mine = -torch.rand(10) - 0.01
    m.log_decay.copy_(mine)
    for cast in (m.bfloat16, m.half, m.double, m.float, lambda: m.to(torch.bfloat16), lambda: m.to("cpu")):
        cast()
        assert m.log_decay.dtype == torch.float32 and torch.equal(m.log_decay, mine)
    net = torch.nn.Sequential(copy.deepcopy(m)).double()
    assert net[0].q.dtype == torch.float64 and torch.equal(net[0].log_decay, mine)
    net.to("meta", torch.bfloat16)
    assert net[0].log_decay.is_meta and net[0].log_decay.dtype == torch.float32
    assert "log_decay" in dict(net[0].named_buffers()) and "log_decay" not in net[0].state_dict()


def test_rates_from_half_to_a_64th():
    m = RoundMemory(96, 3, 2)
    want = torch.log1p(-torch.exp2(-torch.tensor([1.0, 3.5, 6.0], dtype=torch.float64))).float()
    assert torch.equal(m.log_decay.view(2, 3), want.expand(2, 3))
