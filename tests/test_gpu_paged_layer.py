"""The layer's decode() over a paged cache: lengths past the cache's room, positions
past the rotary table."""
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


def test_positions_past_the_table():
    # known on the host: a full cache of more room than the table; else NaN, of such tokens alone
    m = layer(torch.float32, rotary_dim=64, max_positions=40)
    far = layer(torch.float32, rotary_dim=64, max_positions=100)
    far.load_state_dict(m.state_dict())
    table = ints([[2, 0, 4], [5, 1, 3]])
    start = randn(6, 16, 4, 64, seed=3), randn(6, 16, 4, 64, seed=4)
    x = randn(2, 3, 256, seed=5)
    with pytest.raises(ValueError, match="max_positions"):
        m.decode(x, *start, None, table)
    pools = [tuple(t.clone() for t in start) for _ in range(2)]
    # places 38, 39 | 40 of the first sequence and all of the second one
    o, want = (a.decode(x, *p, ints([41, 20]), table) for a, p in zip((m, far), pools))
    assert o[0, 2].isnan().all()
    assert torch.equal(o[0, :2], want[0, :2]) and torch.equal(o[1], want[1])
    # a sequence that is cut back to where it ended is what it was
    y = randn(2, 1, 256, seed=6)
    o, want = (a.decode(y, *p, ints([40, 21]), table) for a, p in zip((m, far), pools))
    assert torch.equal(o, want)
