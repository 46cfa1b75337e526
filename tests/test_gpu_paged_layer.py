"""The layer's decode() over a paged cache: lengths past the cache's room, positions
past the rotary table, trees of drafted tokens, steps captured and replayed."""
import pytest
import torch

import flash_attention_v100 as fa
import paged_oracle as po

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


@pytest.mark.parametrize("dt,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("kw", [{}, {"rotary_dim": 32}, {"rotary_dim": 64, "rotary_interleaved": True, "softcap": 5.0},
                                {"rotary_dim": 64, "distance_bias": True}])
@pytest.mark.parametrize("batch_first", [True, False])
def test_layer_decodes_a_tree(dt, tol, kw, batch_first):
    # each node is what the causal layer computes at the end of the context and the node's
    # ancestors: the same sums in another order.  float32: outputs near 1 of 256 products, 2^-24
    # each way a few times; bf16: projections rounded to 2^-8 of values near 1, in both.
    m = layer(dt, batch_first=batch_first, **kw)
    turn = lambda t: t if batch_first else t.transpose(0, 1)  # noqa: E731
    N, start = 40, [30, 0, 77]
    par = [po.draw_tree(po.rng("layer", b), N) for b in range(3)]
    sees = [po.ancestors(r) for r in par]
    text = randn(3, 77, 256, seed=7, dt=dt)
    x = randn(3, N, 256, seed=8, dt=dt)
    table = ints(po.draw_table(po.rng("layer"), [n + N for n in start], 16, 8, 24))
    kc, vc = (torch.full((24, 16, 4, 64), float("nan"), dtype=dt, device=DEV) for _ in range(2))
    left = torch.zeros_like(text)  # the contexts, each the newest tokens of its row
    for b, n in enumerate(start):
        left[b, 77 - n:] = text[b, :n]
    m.decode(turn(left), kc, vc, ints(start), table)
    pos = ints([[n + len(s) - 1 for s in sees[b]] for b, n in enumerate(start)])
    got = turn(m.decode(turn(x), kc, vc, ints([n + N for n in start]), table, parents=ints(par),
                        positions=pos if m.rotary_dim else None))
    worst = 0.0
    with torch.no_grad():
        for b, n in enumerate(start):
            for i in (0, 1, 7, 20, N - 1):
                want = turn(m(turn(torch.cat([text[b:b + 1, :n], x[b:b + 1, sees[b][i]]], 1)), is_causal=True)[0])[0, -1]
                worst = max(worst, (got[b, i].float() - want.float()).abs().max().item())
    print(f"{dt} {kw}: off by at most {worst:.2e}", flush=True)
    assert worst <= tol


@pytest.mark.parametrize("tree", [False, True])
def test_captured_steps(tree):
    # replays on other lengths, tables and inputs, with eager steps between them, equal the eager step
    N = 5
    m = layer(torch.bfloat16, rotary_dim=64, distance_bias=True)

    def state(seed):
        rng = po.rng("captured", seed)
        lens = [rng.randint(0, 90) for _ in range(3)] + [100]  # the last one past the room
        s = {"x": randn(4, N, 256, seed=seed, dt=torch.bfloat16), "kc": randn(24, 16, 4, 64, seed=seed + 10, dt=torch.bfloat16),
             "vc": randn(24, 16, 4, 64, seed=seed + 20, dt=torch.bfloat16), "lens": ints(lens),
             "table": ints(po.draw_table(rng, [96] * 4, 16, 6, 24))}
        if tree:
            par = [po.draw_tree(rng, N) for _ in range(4)]
            s["par"] = ints(par)
            s["pos"] = ints([[min(n, 96) - N + len(a) - 1 for a in po.ancestors(r)] for n, r in zip(lens, par)])
        return s

    def step(s):
        return m.decode(s["x"], s["kc"], s["vc"], s["lens"], s["table"], parents=s.get("par"), positions=s.get("pos"))

    st = state(1)
    step(state(1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(st)
    for seed in (1, 2, 3, 2):
        fresh = state(seed)
        for name in st:
            st[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, st["kc"], st["vc"])]
        want = (step(fresh), fresh["kc"], fresh["vc"])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed
