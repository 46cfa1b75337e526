"""Calls of the operators around attention at the edge of what they document: tokens
that keep their bits, forward-mode derivatives, empty sides, layers that were used
without gradients first."""
import math

import pytest
import torch

import flash_attention_v100 as fa
from ops_edges_oracle import DEV, DT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 16), (33, 6), (31, 30)])
def test_tokens_at_negative_positions_keep_their_bits(D, R, inter, dt):
    B, S, H = 2, 20, 3
    x = torch.randn(B, S, H, D, generator=torch.Generator("cpu").manual_seed(5)).to(DT[dt]).to(DEV)
    pos = torch.arange(S, device=DEV).repeat(B, 1)
    pos[0, 3:9] = -1
    pos[1] = -7
    out = pos < 0
    vals = torch.tensor([math.inf, -0.0, 1.0, math.nan, -math.inf, 0.0, -2.0], device=DEV).to(DT[dt])
    pad = vals[torch.arange(H * D, device=DEV) % 7].view(H, D)
    x[out] = pad
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    table = fa.rotary_table_v100(64, R, device=DEV)
    before = x.view(bits).clone()
    x.requires_grad_(True)
    y = fa.rotary_embedding_v100(x, None, table, pos, interleaved=inter)
    assert torch.equal(y.detach().view(bits)[out], before[out])
    g, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(g.view(bits)[out], before[out])
    x = x.detach().clone()
    z = fa.rotary_embedding_v100(x, None, table, pos, interleaved=inter, inplace=True)
    assert z is x or z.data_ptr() == x.data_ptr()
    assert torch.equal(x.view(bits), y.detach().view(bits))
