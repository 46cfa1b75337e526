"""flash_attention_v100_paged in units of 128 and 256 rows, whose waves share tiles of
keys: caps, slopes, pages that are none, infinities and NaN in places that a row does not
see, rows of tokens; float32 over columns that head dims from 65 to 96 do not have; one
sequence in hundreds of parts."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo
import paged_oracle as po
from test_gpu_paged import make, run

pytestmark = pytest.mark.gpu
DEV = "cuda"

# lengths whose rows a wave's keys end in, of 64 tokens on 32 and 8 heads: room for 320 keys
# (128 rows, each sequence whole), for 1280 (128 rows, shared) and for 8192 (head dims past 64: 256 rows, shared)
SHORT = [64, 300, 299, 65, 0, 128, 192, 256, 257, 31, 100, 320, 270, 64, 127, 129]
SHARED = [1280, 1000, 64, 700, 0, 129, 1279, 517]
LONG = [8192, 100, 0, 4000, 64, 65, 700, 2500, 1, 3000]
UNITS = {"128": (SHORT, 320), "128 shared": (SHARED, 1280), "256 shared": (LONG, 8192)}
N, H, HKV = 64, 32, 8


def case(units, dt, D, size=16, paged=True, seed=0):
    lens, room = UNITS[units]
    return lens, make(lens, N, room // size if paged else 1, size if paged else room, H, HKV, D, dt, seed=D + seed, paged=paged)


def trees(lens, tree, seed):
    return [po.draw_tree(po.rng(seed, b), N) for b in range(len(lens))] if tree else None


def slopes(B=None):
    s = torch.exp2(-torch.arange(1, H + 1, device=DEV).float() / 4)
    return s if B is None else s * torch.rand(B, H, generator=torch.Generator("cpu").manual_seed(1)).to(DEV)


@pytest.mark.parametrize("units,dt,D", [("128", "bf16", 128), ("128", "fp16", 64), ("128 shared", "fp16", 128),
                                        ("128 shared", "bf16", 32), ("256 shared", "bf16", 128), ("256 shared", "fp16", 96)])
@pytest.mark.parametrize("tree", [False, True])
def test_cap_and_slopes(units, dt, D, tree):
    lens, t = case(units, dt, D)
    par = trees(lens, tree, "rules")
    for label, kw in (("cap", {"softcap": 3.0, "scale": 0.3}), ("wide cap", {"softcap": 1000.0}), ("slopes", {"distance_slopes": slopes()}),
                      ("both, by sequence", {"softcap": 5.0, "distance_slopes": slopes(len(lens))}),
                      ("wide cap and slopes", {"softcap": 500.0, "distance_slopes": slopes()})):
        run(*t[:3], lens, t[3], f"{units} {dt} D={D} tree={tree} {label}", par, **kw)


@pytest.mark.parametrize("units,dt,D", [("128", "bf16", 128), ("128 shared", "fp16", 64), ("256 shared", "fp16", 128)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("size", [16, 64])
def test_pages_that_are_none(units, dt, D, tree, size):
    lens, t = case(units, dt, D, size, seed=1)
    rng, P = po.rng("none", size), t[1].shape[0]
    table = [r[:] for r in t[3]]
    for b, n in enumerate(lens):
        cols = range(-(-n // size))
        for c in rng.sample(cols, min(len(cols), 1 + len(cols) // 5)) if b % 3 != 1 else ():
            table[b][c] = rng.choice([-1, P, 2 ** 31 - 1, -(2 ** 31)])
    par = trees(lens, tree, "none")
    run(*t[:3], lens, table, f"{units} pages that are none", par)
    run(*t[:3], lens, table, f"{units} pages that are none, rules", par, softcap=4.0, distance_slopes=slopes())
    o, lse = run(*t[:3], lens, [[-1] * len(r) for r in table], f"{units} no pages at all", par)
    assert not o.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("units,dt,D", [("128", "fp16", 128), ("128 shared", "bf16", 64), ("256 shared", "bf16", 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_infinities_of_nodes_that_others_do_not_see(units, dt, D, bad):
    # node 20 of each tree (a leaf beside 63 others): what sees it is no number, all else stays
    lens, t = case(units, dt, D, seed=2)
    par = [[p if p != 20 else 19 for p in r] for r in trees(lens, True, "hidden")]
    sees = [[20 in s for s in po.ancestors(r)] for r in par]
    assert all(sum(s) == 1 for s in sees)
    ref = po.attention(*t[:3], lens, t[3], par, 6.0, slopes())
    kc, vc = t[1].clone(), t[2].clone()
    for b, n in enumerate(lens):
        if n - N + 20 >= 0:
            p, r = po.place(t[3], b, n - N + 20, 16)
            vc[p, r, :, ::3] = bad
            kc[p, r, :, 5] = bad
    ints = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
    o, lse = fa.flash_attention_v100_paged(t[0], kc, vc, ints(lens), ints(t[3]), parents=ints(par), softcap=6.0,
                                           distance_slopes=slopes(), return_softmax_lse=True)
    others = [i for i in range(N) if i != 20]
    oo.check({"o": o[:, others], "lse": lse[:, :, others]},
             {"o": tuple(x[:, others] for x in ref["o"]), "lse": tuple(x[:, :, others] for x in ref["lse"])}, ["o", "lse"], units)
    for b, n in enumerate(lens):
        if n - N + 20 >= 0:
            assert o[b, 20, :, ::3].isnan().any() or (o[b, 20, :, ::3] == bad).any()


@pytest.mark.parametrize("units,dt,D", [("128", "bf16", 128), ("128 shared", "fp16", 128), ("256 shared", "bf16", 96)])
def test_infinities_behind_the_chain(units, dt, D):
    # the last 20 tokens are no numbers to those before them
    lens, t = case(units, dt, D, seed=3)
    ref = po.attention(*t[:3], lens, t[3], None, 0.0, slopes())
    kc, vc = t[1].clone(), t[2].clone()
    for b, n in enumerate(lens):
        for x in range(max(0, n - 20), n):
            p, r = po.place(t[3], b, x, 16)
            vc[p, r, :, x % 7::7] = (math.inf, -math.inf, math.nan)[x % 3]
            kc[p, r, :, x % D] = (math.nan, math.inf, -math.inf)[x % 3]
    ints = lambda x: torch.tensor(x, device=DEV)  # noqa: E731
    o, lse = fa.flash_attention_v100_paged(t[0], kc, vc, ints(lens), ints(t[3]), distance_slopes=slopes(), return_softmax_lse=True)
    oo.check({"o": o[:, :-20], "lse": lse[:, :, :-20]},
             {"o": tuple(x[:, :-20] for x in ref["o"]), "lse": tuple(x[:, :, :-20] for x in ref["lse"])}, ["o", "lse"], units)


@pytest.mark.parametrize("units,dt,D", [("128", "fp16", 128), ("128 shared", "bf16", 64), ("256 shared", "fp16", 128)])
@pytest.mark.parametrize("tree", [False, True])
def test_rows_of_tokens(units, dt, D, tree):
    lens, t = case(units, dt, D, paged=False, seed=4)
    par = trees(lens, tree, "rows")
    run(*t[:3], lens, None, f"{units} rows", par)
    run(*t[:3], lens, None, f"{units} rows, rules", par, softcap=30.0, distance_slopes=slopes())
    clean = [torch.nan_to_num(x) for x in t[:3]]
    run(*clean, None, None, f"{units} rows, all filled", par)


@pytest.mark.parametrize("D", [68, 80, 96])
@pytest.mark.parametrize("n,tree", [(1, False), (33, False), (40, True)])
def test_float32_of_three_quarters_of_the_columns(D, n, tree):
    # lengths far apart, so that units are shared
    lens = [3000, 130, 0, 1450, 1, 517]
    t = make(lens, n, 188, 16, 8, 2, D, "fp32", seed=D)
    par = [po.draw_tree(po.rng(n, b), n) for b in range(len(lens))] if tree else None
    run(*t[:3], lens, t[3], f"D={D} N={n}", par)
    run(*t[:3], lens, t[3], f"D={D} N={n} rules", par, softcap=20.0, distance_slopes=slopes()[:8].clone())
    kc, vc = t[1].clone(), t[2].clone()
    ref = po.attention(*t[:3], lens, t[3], par)
    for b, m in enumerate(lens):  # the newest token is no number (a leaf of the tree)
        if m:
            p, r = po.place(t[3], b, m - 1, 16)
            kc[p, r, :, D - 1] = vc[p, r, :, ::5] = math.inf
    ints = lambda x: None if x is None else torch.tensor(x, device=DEV)  # noqa: E731
    o, lse = fa.flash_attention_v100_paged(t[0], kc, vc, ints(lens), ints(t[3]), parents=ints(par), return_softmax_lse=True)
    if n > 1:
        oo.check({"o": o[:, :-1], "lse": lse[:, :, :-1]},
                 {"o": tuple(x[:, :-1] for x in ref["o"]), "lse": tuple(x[:, :, :-1] for x in ref["lse"])}, ["o", "lse"], f"D={D}")


@pytest.mark.parametrize("dt,D,B,room", [("fp16", 32, 1, 1 << 17), ("bf16", 128, 1, 40000), ("fp32", 64, 2, 50000)])
def test_hundreds_of_parts(dt, D, B, room):
    # one KV head and one unit: 512, 157 and about 390 parts, which the join's waves take in several turns
    lens = [room - 5] + [3] * (B - 1)
    t = make(lens, 1, -(-room // 64), 64, 4, 1, D, dt, seed=5)
    run(*t[:3], lens, t[3], f"{dt} {room}")
    run(*t[:3], lens, t[3], f"{dt} {room} slopes", distance_slopes=torch.tensor([0.5, 1e-3, 1e-5, -1e-5], device=DEV))
