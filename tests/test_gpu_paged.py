"""flash_attention_v100_paged against the 64-bit oracle: chains and trees of new
tokens, pages and rows of tokens, what hidden places hold."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo
import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(lens, N, M, size, H, Hkv, D, dt, seed=0, paged=True, spare=3):
    """(q, k pool, v pool, page table as lists or None); unused places hold NaN."""
    g = torch.Generator("cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DT[dt]).to(DEV)  # noqa: E731
    B = len(lens)
    used = sum(-(-max(0, n) // size) for n in lens)
    P = used + spare if paged else B
    table = po.draw_table(po.rng("table", seed), [max(0, n) for n in lens], size, M, P) if paged else None
    q, kc, vc = r(B, N, H, D), r(P, size, Hkv, D), r(P, size, Hkv, D)
    filled = torch.zeros(P, size, dtype=torch.bool)
    for b, n in enumerate(lens):
        for x in range(n):
            filled[po.place(table, b, x, size)] = True
    for t in (kc, vc):
        t[~filled.to(DEV)] = math.nan
    return q, kc, vc, table


def run(q, kc, vc, lens, table, label, parents=None, dtype=torch.int32, **kw):
    ints = lambda x: None if x is None else torch.tensor(x, dtype=dtype, device=DEV)  # noqa: E731
    o, lse = fa.flash_attention_v100_paged(q, kc, vc, ints(lens), ints(table), parents=ints(parents),
                                           return_softmax_lse=True, **kw)
    ref = po.attention(q, kc, vc, lens, table, parents, kw.get("softcap") or 0.0, kw.get("distance_slopes"),
                       kw.get("scale"))
    oo.check({"o": o, "lse": lse}, ref, ["o", "lse"], label)
    return o, lse


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("N,tree", [(1, False), (5, False), (13, True)])
def test_types_dims(dt, D, N, tree):
    lens = [200, 129, 64, N, N - 1, 0, 33]
    t = make(lens, N, 13, 16, 8, 2, D, dt, seed=D + N)
    rng = po.rng(D, N)
    parents = [po.draw_tree(rng, N) for _ in lens] if tree else None
    o, lse = run(*t[:3], lens, t[3], f"{dt} D={D} N={N}", parents)
    assert not o[5].any() and (lse[5] == -math.inf).all()


@pytest.mark.parametrize("size", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("N", [1, 7])
def test_page_sizes(size, N):
    lens = [1000, 16, 17, 31, 513, 768, N]
    t = make(lens, N, -(-1000 // size), size, 4, 2, 64, "bf16", seed=size)
    run(*t[:3], lens, t[3], f"size {size}")
    run(*t[:3], lens, t[3], f"size {size} tree", po.draw_tree(po.rng(size), N))


@pytest.mark.parametrize("room", [1, 5, 100, 1003])
def test_rows_of_tokens(room):
    lens = [room, max(1, room // 2), 1]
    N = min(3, room)
    t = make(lens, N, 1, room, 6, 3, 128, "fp16", seed=room, paged=False)
    run(*t[:3], lens, None, f"room {room}")
    run(*t[:3], lens, None, f"room {room} tree", po.draw_tree(po.rng(room), N))
    clean = [torch.nan_to_num(x) for x in t[:3]]
    run(*clean, None, None, f"room {room} all filled")


@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (12, 4), (32, 8), (40, 1), (64, 8)])
@pytest.mark.parametrize("N", [1, 9])
def test_heads(H, Hkv, N):
    lens = [300, 77]
    t = make(lens, N, 10, 32, H, Hkv, 64, "bf16", seed=H + Hkv)
    run(*t[:3], lens, t[3], f"{H} on {Hkv}", po.draw_tree(po.rng(H), N) if N > 1 else None)


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("fp16", 64), ("fp32", 128), ("fp32", 64)])
@pytest.mark.parametrize("N,tree", [(1, False), (64, True), (100, False)])
def test_units_shared_by_workgroups(dt, D, N, tree):
    # lengths far apart, so that workgroups end inside units and begin others
    lens = [6000, 130, 0, 2900, 1, 517]
    t = make(lens, N, 48, 128, 8, 2, D, dt, seed=5)
    rng = po.rng(N, D)
    run(*t[:3], lens, t[3], f"{dt} {N}", [po.draw_tree(rng, N) for _ in lens] if tree else None)


@pytest.mark.parametrize("dt,D,N", [("bf16", 128, 1), ("fp16", 64, 15), ("fp32", 64, 3), ("fp32", 128, 1)])
def test_units_in_many_parts(dt, D, N):
    # one long sequence beside a short one and an empty one: more than 40 parts of a unit
    lens = [12000 + N] if dt != "fp32" else [11000, 0]
    t = make(lens, N, 768, 16, 4, 2, D, dt, seed=D + N)
    run(*t[:3], lens, t[3], f"{dt} D={D} N={N}")


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("fp16", 64), ("bf16", 32)])
@pytest.mark.parametrize("tree", [False, True])
def test_wide_units_of_short_sequences(dt, D, tree):
    N, lens = 64, [64, 300, 299, 65, 0, 128, 192, 256, 257, 31, 100, 320, 270, 64, 127, 129]
    t = make(lens, N, 20, 16, 32, 8, D, dt, seed=D)
    par = [po.draw_tree(po.rng("short", b), N) for b in range(len(lens))] if tree else None
    run(*t[:3], lens, t[3], f"{dt} D={D} tree={tree}", par)


@pytest.mark.parametrize("dt,D,tree", [("bf16", 128, True), ("fp16", 96, False)])
def test_units_of_256_rows(dt, D, tree):
    # room that makes the units the widest, in sequences of all lengths
    N, lens = 64, [8192, 100, 0, 4000, 64, 65, 700, 2500, 1, 3000]
    t = make(lens, N, 512, 16, 32, 8, D, dt, seed=D)
    par = [po.draw_tree(po.rng("wide", b), N) for b in range(len(lens))] if tree else None
    run(*t[:3], lens, t[3], f"{dt} D={D} tree={tree}", par)


def test_many_sequences():
    rng = po.rng("many")
    lens = [rng.randint(0, 700) for _ in range(150)]
    lens[149] = 700
    t = make(lens, 1, 44, 16, 4, 1, 64, "bf16", seed=6)
    run(*t[:3], lens, t[3], "150 sequences")
    t = make(lens, 4, 44, 16, 4, 1, 64, "bf16", seed=7)
    run(*t[:3], lens, t[3], "150 trees", [po.draw_tree(rng, 4) for _ in lens])


@pytest.mark.parametrize("B,N,dt,D,room", [(150, 1, "bf16", 64, 4800), (130, 4, "fp32", 32, 1600), (70, 64, "fp16", 128, 1152)])
def test_many_sequences_share_units(B, N, dt, D, room):
    # more sequences than lanes, some much longer than the others
    rng = po.rng("share", B)
    lens = [rng.randint(0, 300) for _ in range(B)]
    for b in (3, 64, B - 1):
        lens[b] = rng.randint(room * 3 // 4, room)
    t = make(lens, N, room // 16, 16, 4, 1, D, dt, seed=B)
    run(*t[:3], lens, t[3], f"{B} sequences", [po.draw_tree(rng, N) for _ in lens] if N > 1 else None)


@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 64, 65, 128, 256])
def test_trees(N):
    lens = [N + 45, N, N + 700, max(0, N - 2)]
    t = make(lens, N, -(-(N + 700) // 16), 16, 4, 2, 64, "fp16", seed=N)
    rng = po.rng("trees", N)
    trees = [po.draw_tree(rng, N, depth=N) for _ in lens]
    run(*t[:3], lens, t[3], "own trees", trees)
    run(*t[:3], lens, t[3], "chain as a tree", list(range(-1, N - 1)))
    run(*t[:3], lens, t[3], "no token follows another", [-1] * N)
    chain = fa.flash_attention_v100_paged(*t[:3], torch.tensor(lens, device=DEV), torch.tensor(t[3], device=DEV))
    assert not chain.isnan().any()


def test_padding_and_what_is_no_tree():
    N = 40
    lens = [300, 45, 40]
    t = make(lens, N, 19, 16, 4, 2, 64, "bf16", seed=8)
    rows = [[-1, 0, 0, 1, -2, 4, 3, 7, 9, 2 ** 31 - 1, -(2 ** 31)] + [5] * (N - 11),  # padding, its followers, itself, a later one
            [-2] * N, [i for i in range(N)]]
    o, lse = run(*t[:3], lens, t[3], "padding", rows)
    assert not o[1:].any() and (lse[1:] == -math.inf).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("tree", [False, True])
def test_cap_slopes_scale(dt, tree):
    N, lens = 11, [400, 90, 11, 7, 0]
    t = make(lens, N, 25, 16, 8, 4, 128, dt, seed=9)
    par = [po.draw_tree(po.rng(b), N) for b in range(5)] if tree else None
    sl = torch.exp2(-torch.arange(1, 9, device=DEV).float())
    run(*t[:3], lens, t[3], "cap", par, softcap=3.0, scale=0.3)
    run(*t[:3], lens, t[3], "wide cap", par, softcap=1000.0)
    run(*t[:3], lens, t[3], "slopes", par, distance_slopes=sl)
    run(*t[:3], lens, t[3], "both, by sequence", par, softcap=3.0, distance_slopes=sl * torch.rand(5, 8, device=DEV))


@pytest.mark.parametrize("N", [3, 70, 200])
def test_slopes_over_tile_borders(N):
    # the new tokens begin at every place of a tile
    lens = [N + x for x in (0, 1, 15, 16, 31, 32, 33, 47, 63, 64, 65, 95)]
    t = make(lens, N, -(-(N + 95) // 16), 16, 4, 2, 32, "fp32", seed=N)
    par = [po.draw_tree(po.rng(N, b), N) for b in range(len(lens))]
    sl = torch.tensor([0.5, 0.1, 0.03, -0.02], device=DEV)
    run(*t[:3], lens, t[3], "slopes", par, distance_slopes=sl)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("N", [6, 60])
def test_hidden_infinities(dt, tree, N):
    # the newest token's own key and value are no numbers: nothing else changes
    lens = [200, 97, N]
    t = make(lens, N, 13, 16, 4, 2, 64, dt, seed=10)
    par = [po.draw_tree(po.rng(b), N - 1) + [0] for b in range(3)] if tree else None
    ints = lambda x: None if x is None else torch.tensor(x, device=DEV)  # noqa: E731
    args = (ints(lens), ints(t[3]))
    want, wlse = fa.flash_attention_v100_paged(*t[:3], *args, parents=ints(par), return_softmax_lse=True)
    for bad in (math.nan, math.inf, -math.inf):
        kc, vc = t[1].clone(), t[2].clone()
        for b, n in enumerate(lens):
            p, r = po.place(t[3], b, n - 1, 16)
            vc[p, r, :, ::3] = bad
            kc[p, r, :, 5] = bad
        o, lse = fa.flash_attention_v100_paged(t[0], kc, vc, *args, parents=ints(par), return_softmax_lse=True)
        ref = po.attention(*t[:3], lens, t[3], par)
        oo.check({"o": o[:, :-1], "lse": lse[:, :, :-1]},
                 {"o": tuple(x[:, :-1] for x in ref["o"]), "lse": tuple(x[:, :, :-1] for x in ref["lse"])}, ["o", "lse"], str(bad))
        assert o[:, -1].isnan().any()
    # a value alone that is infinite stays infinite where it is seen
    vc = t[2].clone()
    for b, n in enumerate(lens):
        p, r = po.place(t[3], b, n - 1, 16)
        vc[p, r, :, 7] = math.inf
    o = fa.flash_attention_v100_paged(t[0], t[1], vc, *args, parents=ints(par))
    assert (o[:, -1, :, 7] == math.inf).all() and torch.isfinite(o[:, :-1]).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_hidden_infinities_of_waves_of_one_token(dt):
    # 64 heads of a KV head: all rows of a wave are one token's, and other waves of the unit see more
    N, lens = 8, [2048, 1000, 2047, 8, 1999, 64, 1500, 777, 2048, 130, 1, 0, 1024, 2048, 31, 1600]
    t = make(lens, N, 128, 16, 64, 1, 32, dt, seed=11)
    kc, vc = t[1].clone(), t[2].clone()
    for b, n in enumerate(lens):
        if n:
            p, r = po.place(t[3], b, n - 1, 16)
            kc[p, r, :, 5] = vc[p, r, :, ::3] = math.inf
    ints = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
    o, lse = fa.flash_attention_v100_paged(t[0], kc, vc, ints(lens), ints(t[3]), return_softmax_lse=True)
    ref = po.attention(*t[:3], lens, t[3])
    oo.check({"o": o[:, :-1], "lse": lse[:, :, :-1]},
             {"o": tuple(x[:, :-1] for x in ref["o"]), "lse": tuple(x[:, :, :-1] for x in ref["lse"])}, ["o", "lse"], dt)


def test_pages_that_are_none():
    N, lens = 4, [200, 64, 130]
    t = make(lens, N, 13, 16, 4, 2, 64, "bf16", seed=12)
    table = [r[:] for r in t[3]]
    table[0][3], table[0][5], table[1][1], table[2][8] = -1, t[1].shape[0], 2 ** 31 - 1, -7
    for par in (None, [-1, 0, 0, 1]):
        run(*t[:3], lens, table, "no page", par)
        o, lse = run(*t[:3], lens, [[-1] * 13] * 3, "no pages at all", par)
        assert not o.any() and (lse == -math.inf).all()
    run(*t[:3], lens, [[2 ** 40 if p < 0 else p for p in r] for r in t[3]], "64-bit numbers", dtype=torch.int64)


def test_lengths_past_the_room():
    t = make([64, 64], 2, 4, 16, 4, 2, 64, "bf16", seed=13)
    want = run(*t[:3], [64, 64], t[3], "full")
    got = fa.flash_attention_v100_paged(*t[:3], torch.tensor([10 ** 6, 2 ** 40], device=DEV), torch.tensor(t[3], device=DEV))
    assert torch.equal(got, want[0])
    got, lse = fa.flash_attention_v100_paged(*t[:3], torch.tensor([-5, -2 ** 40], device=DEV), torch.tensor(t[3], device=DEV),
                                             return_softmax_lse=True)
    assert not got.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("D,dt", [(96, "bf16"), (80, "fp16"), (8, "bf16"), (36, "fp32"), (100, "fp32"), (40, "fp16")])
def test_head_dims_between(D, dt):
    lens = [150, 33]
    t = make(lens, 3, 10, 16, 4, 2, D, dt, seed=D)
    run(*t[:3], lens, t[3], f"D={D}", [-1, 0, 0])


def test_strides_and_types_of_integers():
    N, lens, size, Hkv, D = 3, [120, 40], 16, 2, 64
    q, kc, vc, table = make(lens, N, 8, size, 4, Hkv, D, "bf16", seed=14)
    ints = lambda x, d=torch.int32: torch.tensor(x, device=DEV, dtype=d)  # noqa: E731
    par = [-1, 0, 0]
    want = fa.flash_attention_v100_paged(q, kc, vc, ints(lens), ints(table), parents=ints(par))
    k2 = kc.transpose(1, 2).contiguous().transpose(1, 2)               # heads first in a page
    v2 = torch.stack([vc, vc], 1)[:, 1]                                # a page of two pools' rows
    q2 = torch.cat([q, q], -1)[..., :D]
    t2 = ints(table, torch.int64).t().contiguous().t()                 # columns first
    p2 = ints([par, par], torch.int64)
    got = fa.flash_attention_v100_paged(q2, k2, v2, ints(lens, torch.int64), t2, parents=p2)
    assert torch.equal(got, want)
    assert torch.equal(fa.flash_attention_v100_paged(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, ints(lens),
                                                     ints(table), parents=ints(par).expand(2, N)), want)


def test_pool_past_32_bits():
    # pages beyond 4 GiB of a pool, and a row stride that spans several heads' rows
    size, Hkv, D = 16, 8, 128
    P = (5 << 30) // (size * Hkv * D * 2)
    kc = torch.zeros(P, size, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    lens, N = [100, 40], 2
    small = make(lens, N, 7, size, 8, Hkv, D, "bf16", seed=15)
    far = [[P - 1 - p if p >= 0 else -1 for p in r] for r in small[3]]
    n = small[1].shape[0]
    kc[P - n:], vc[P - n:] = small[1].flip(0), small[2].flip(0)
    ints = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
    want = fa.flash_attention_v100_paged(*small[:3], ints(lens), ints(small[3]))
    assert torch.equal(fa.flash_attention_v100_paged(small[0], kc, vc, ints(lens), ints(far)), want)


def test_rows_of_millions_of_tokens():
    # the last tokens of rows longer than a page may be: what they hold decides
    size, D, N = 2 ** 21 + 16, 32, 2
    g = torch.Generator(DEV).manual_seed(18)
    kc = torch.zeros(2, size, 1, D, dtype=torch.float16, device=DEV)
    vc = torch.zeros_like(kc)
    q = torch.zeros(2, N, 1, D, dtype=torch.float16, device=DEV)
    q[..., 0] = 30.0
    kc[:, -40:, :, 0] = 3.0                                    # e^90 against e^0 of 2^21 others
    vc[:, -40:] = torch.randn(2, 40, 1, D, generator=g, device=DEV).half()
    o = fa.flash_attention_v100_paged(q, kc, vc, scale=1.0)
    for i in range(N):
        want = vc[:, size - 40:size - N + i + 1, 0].double().mean(1)
        # the products and sums of up to 40 probabilities (one each, e^-90 times 2^21 beside them) in fp16 and float32
        bound = want.abs() * 2.0 ** -11 + vc[:, -40:, 0].double().abs().mean(1) * (2.0 ** -11 + 41 * 2.0 ** -24) + 2.0 ** -25
        assert ((o[:, i, 0].double() - want).abs() <= bound).all()


def test_empty_sides():
    q, kc, vc, table = make([16, 5], 2, 1, 16, 4, 2, 64, "bf16", seed=16)
    ints = lambda x: torch.tensor(x, device=DEV, dtype=torch.int32)  # noqa: E731
    assert fa.flash_attention_v100_paged(q[:0], kc, vc, ints([]), ints(table)[:0]).shape == (0, 2, 4, 64)
    assert fa.flash_attention_v100_paged(q[:, :0], kc, vc, ints([16, 5]), ints(table)).shape == (2, 0, 4, 64)
    for args in ((kc, vc, ints([16, 5]), ints(table)[:, :0]), (kc[:0], vc[:0], ints([16, 5]), ints(table)),
                 (kc[:2, :0], vc[:2, :0], ints([3, 3]), None)):
        o, lse = fa.flash_attention_v100_paged(q, *args, return_softmax_lse=True)
        assert not o.any() and (lse == -math.inf).all()


def test_equal_to_scored_attention():
    # a chain over a row of tokens is what the cache attention of single tokens computes
    q, kc, vc, _ = make([500, 123, 17], 5, 1, 500, 8, 2, 128, "bf16", seed=17, paged=False)
    lens = torch.tensor([500, 123, 17], device=DEV)
    ref = po.attention(q, kc, vc, lens.tolist(), None)
    a = fa.flash_attention_v100_paged(q, kc, vc, lens, return_softmax_lse=True)
    b = fa.flash_attention_v100_scored(q, kc, vc, causal=True, key_lengths=lens, query_offsets=lens - 5,
                                       return_softmax_lse=True)
    for x in (a, b):
        oo.check({"o": x[0], "lse": x[1]}, ref, ["o", "lse"], "")


def test_refuses_gradients():
    q, kc, vc, table = make([16], 1, 1, 16, 2, 2, 64, "bf16")
    q.requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no_grad"):
        fa.flash_attention_v100_paged(q, kc, vc, None, torch.tensor(table, device=DEV))
    with torch.no_grad():
        assert not fa.flash_attention_v100_paged(q, kc, vc, None, torch.tensor(table, device=DEV)).requires_grad
