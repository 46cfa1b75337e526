"""flash_attention_v100_shared_prefix against the 64-bit oracle over the
concatenated keys."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(B, Sq, P, Sk, H, Hkv, D, dt, seed=0):
    g = torch.Generator("cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DT[dt]).to(DEV)  # noqa: E731
    return r(B, Sq, H, D), r(P, Hkv, D), r(P, Hkv, D), r(B, Sk, Hkv, D), r(B, Sk, Hkv, D)


def oracle(q, kp, vp, k, v, lens, softcap=0.0, slopes=None, scale=None):
    B, Sq = q.shape[:2]
    P, Sk = kp.shape[0], k.shape[1]
    kc, vc = (torch.cat([a.unsqueeze(0).expand(B, *a.shape), b], 1) for a, b in ((kp, k), (vp, v)))
    own = lens.long().clamp(0, Sk).view(B, 1) - Sq + torch.arange(Sq, device=DEV)  # (B, Sq)
    j = torch.arange(P + Sk, device=DEV) - P
    seen = (j <= own[..., None]) & (own[..., None] >= 0)
    return oo.scored(q, kc, vc, None, scale, softcap, slopes, 0, seen, kpos=j, qpos=own)


def run(t, lens, label, **kw):
    o, lse = fa.flash_attention_v100_shared_prefix(*t, key_lengths=lens, return_softmax_lse=True, **kw)
    full = lens if lens is not None else torch.full((t[0].shape[0],), t[3].shape[1], device=DEV)
    clean = [torch.nan_to_num(x) for x in t]
    ref = oracle(*clean, full, kw.get("softcap") or 0.0, kw.get("distance_slopes"), kw.get("scale"))
    oo.check({"o": o, "lse": lse}, ref, ["o", "lse"], label)
    return o, lse


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Sq", [1, 3])
def test_types_dims(dt, D, Sq):
    t = make(6, Sq, 333, 70, 8, 2, D, dt, seed=D + Sq)
    lens = torch.tensor([70, 64, 33, Sq, Sq - 1, 0], dtype=torch.int32, device=DEV)
    for b in range(6):  # behind the filled keys there may be anything
        t[3][b, int(lens[b]):] = math.nan
        t[4][b, int(lens[b]):] = math.inf
    t[4].nan_to_num_(nan=math.nan, posinf=math.nan)
    o, lse = run(t, lens, f"{dt} D={D} Sq={Sq}")
    assert not o[5].any() and (lse[5] == -math.inf).all()


@pytest.mark.parametrize("P,Sk,B,Sq,H,Hkv", [(0, 40, 3, 1, 4, 4), (1, 1, 1, 1, 1, 1), (64, 64, 2, 2, 4, 1),
                                             (65, 129, 5, 1, 6, 3), (4097, 3, 40, 1, 16, 4), (700, 900, 2, 7, 32, 2),
                                             (1000, 17, 33, 5, 4, 4)])
def test_sizes(P, Sk, B, Sq, H, Hkv):
    Sq = min(Sq, Sk)
    t = make(B, Sq, P, Sk, H, Hkv, 64, "bf16", seed=P + Sk)
    g = torch.Generator("cpu").manual_seed(7)
    lens = torch.randint(Sq, Sk + 1, (B,), generator=g).to(DEV)
    run(t, lens, f"P={P} Sk={Sk}")
    run(t, None, f"P={P} Sk={Sk} all filled")


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
def test_cap_slopes_scale(dt):
    t = make(4, 2, 500, 90, 8, 4, 128, dt, seed=11)
    lens = torch.tensor([90, 50, 2, 77], dtype=torch.int32, device=DEV)
    sl = torch.exp2(-torch.arange(1, 9, device=DEV).float())
    run(t, lens, "cap", softcap=3.0, scale=0.3)
    run(t, lens, "slopes", distance_slopes=sl)
    run(t, lens, "both, by sequence", softcap=3.0, distance_slopes=sl * torch.rand(4, 8, device=DEV))


@pytest.mark.parametrize("D,dt", [(96, "bf16"), (80, "fp16"), (20, "bf16"), (36, "fp32"), (5, "fp16")])
def test_head_dims_between(D, dt):
    t = make(3, 1, 130, 20, 4, 2, D, dt, seed=D)
    run(t, torch.tensor([20, 7, 1], device=DEV), f"D={D}")


def test_strides():
    B, P, Sk, H, Hkv, D = 3, 200, 50, 4, 2, 64
    t = list(make(B, 1, P, Sk, H, Hkv, D, "bf16", seed=13))
    want = fa.flash_attention_v100_shared_prefix(*t)
    t[1] = t[1].transpose(0, 1).contiguous().transpose(0, 1)          # heads first
    t[2] = torch.cat([t[2], t[2]], -1)[..., :D]                        # rows apart
    t[3] = torch.cat([t[3], t[3]], 1)[:, :Sk]                          # part of a larger cache
    t[0] = t[0].expand(B, 1, H, D)
    assert torch.equal(fa.flash_attention_v100_shared_prefix(*t), want)


def test_equal_to_one_attention_over_all_keys():
    # the single-token form over each sequence's whole keys: the same values, other splits
    B, P, Sk = 4, 600, 60
    t = make(B, 1, P, Sk, 8, 2, 128, "bf16", seed=14)
    lens = torch.tensor([60, 31, 1, 45], device=DEV)
    o = fa.flash_attention_v100_shared_prefix(*t, key_lengths=lens)
    kc, vc = (torch.cat([a.unsqueeze(0).expand(B, *a.shape), b], 1) for a, b in ((t[1], t[3]), (t[2], t[4])))
    o2, lse2 = fa.flash_attention_v100_scored(t[0], kc, vc, causal=True, key_lengths=P + lens,
                                              query_offsets=P + lens - 1, return_softmax_lse=True)
    ref = oracle(*t, lens)
    oo.check({"o": o}, ref, ["o"], "shared")
    oo.check({"o": o2, "lse": lse2}, ref, ["o", "lse"], "one cache")


def test_refuses_gradients():
    t = make(2, 1, 10, 5, 2, 2, 64, "bf16")
    t[0].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no_grad"):
        fa.flash_attention_v100_shared_prefix(*t)
    with torch.no_grad():
        assert not fa.flash_attention_v100_shared_prefix(*t).requires_grad


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,Sq", [(3, 1), (33, 1), (9, 5)])
def test_long_prefixes(dt, D, B, Sq):
    # units of 32 and of 128 rows over several parts of a prefix that ends inside a
    # tile, free slots among them
    P, Sk, H, Hkv = 1500, 70, 8, 2
    t = make(B, Sq, P, Sk, H, Hkv, D, dt, seed=21)
    lens = torch.randint(0, Sk + 1, (B,), generator=torch.Generator("cpu").manual_seed(2)).to(DEV)
    lens[B // 2] = 0
    for b in range(B):
        t[3][b, int(lens[b]):] = math.nan
    g = torch.Generator("cpu").manual_seed(3)
    slopes = (0.02 * torch.rand(B, H, generator=g)).to(DEV)
    run(t, lens, f"{dt} {D} {B}x{Sq}")
    run(t, lens, f"{dt} {D} {B}x{Sq} cap, slopes", softcap=12.0, distance_slopes=slopes)
