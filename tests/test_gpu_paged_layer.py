"""The layer's decode() over a paged cache: lengths past the cache's room."""
import pytest
import torch

import flash_attention_v100 as fa

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def layer(dt, seed=0, **kw):
    torch.manual_seed(seed)
    return fa.EnhancedMultiHeadAttention(256, 4, **kw).to(DEV, dt).eval()


def randn(*shape, seed=0, dt=torch.float32):
    return torch.randn(*shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dt).to(DEV)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lengths_past_the_room_count_as_the_room(paged, dtype):
    # in the rows that are written, in what is attended to and in the rotary positions alike
    m = layer(torch.float32, rotary_dim=64)
    room, N = 48, 3
    table = ints([[2, 0, 4], [5, 1, 3]]) if paged else None
    start = randn(*((6, 16) if paged else (2, room)), 4, 64, seed=1)
    x = randn(2, N, 256, seed=2)
    outs = []
    for lens in ([room, room], [room + 5, 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 40]):
        kc, vc = start.clone(), start.flip(0).clone()
        outs.append((m.decode(x, kc, vc, ints(lens, dtype), table), kc, vc))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
