"""Caps far above the scores: for |x| far below the cap the result is that without
one, within bounds that do not grow with the cap.  Small gradients under a cap."""
import pytest
import torch

import flash_attention_v100 as fa
import ops_edges_oracle as eo
import ops_oracle as oo
import test_gpu_scored as ts
from ops_edges_oracle import DEV, make, train

pytestmark = pytest.mark.gpu


WIDE = [257.0, 1e4, 1e6, 1e8, 1e30]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("cap", WIDE)
def test_wide_caps(cap, D, dt):
    q, k, v, do = make(2, 197, 197, 4, 2, D, dt, seed=D)
    train(2 * q, 2 * k, v, do, f"cap {cap} D={D} {dt}", causal=True, softcap=cap)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [1e4, 1e8])
def test_wide_caps_of_other_calls(cap, dt):
    # documents, slopes, and a grid of one group of waves a block
    q, k, v, do = make(2, 150, 150, 2, 1, 64, dt, seed=1)
    docs = (torch.arange(150, device=DEV) // 40).int()
    docs[130:] = -1
    slopes = torch.tensor([0.25, 0.01], device=DEV)
    train(q, k, v, do, "documents", softcap=cap, documents=docs)
    train(q, k, v, do, "slopes", softcap=cap, distance_slopes=slopes)
    q, k, v, do = make(5, 500, 500, 30, 30, 64, dt, seed=2)
    train(q, k, v, do, "one group", softcap=cap, causal=True)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("cap", WIDE)
def test_wide_caps_of_tokens_and_prefixes(cap, dt):
    B, Sk, P, H, Hkv, D = 3, 700, 900, 8, 2, 64
    q, k, v, _ = make(B, 1, Sk, H, Hkv, D, dt, seed=3)
    kp, vp = (t[0] for t in make(1, 1, P, H, Hkv, D, dt, seed=4)[1:3])
    q = 2 * q
    lens = torch.tensor([700, 65, 1], dtype=torch.int32, device=DEV)
    got = dict(zip(("o", "lse"), fa.flash_attention_v100_scored(
        q, k, v, causal=True, softcap=cap, key_lengths=lens, query_offsets=lens - 1, return_softmax_lse=True)))
    seen = oo.seen_mask(B, 1, Sk, True, None, None, None, lens, lens - 1, DEV)
    oo.check(got, eo.scored(q, k, v, None, cap, None, lens - 1, seen, lens), ["o", "lse"], f"tokens {cap} {dt}")
    for n in (P, 300):  # parts that are joined, and one walk
        got = dict(zip(("o", "lse"), fa.flash_attention_v100_shared_prefix(
            q, kp[:n], vp[:n], k[:, :100], v[:, :100], lens.clamp(max=100), softcap=cap, return_softmax_lse=True)))
        cat = lambda a, b: torch.cat([a[:n].expand(B, n, Hkv, D), b[:, :100]], 1)  # noqa: E731
        all_lens = lens.clamp(max=100) + n
        seen = oo.seen_mask(B, 1, n + 100, True, None, None, None, all_lens, all_lens - 1, DEV)
        ref = eo.scored(q, cat(kp, k), cat(vp, v), None, cap, None, all_lens - 1, seen, all_lens)
        oo.check(got, ref, ["o", "lse"], f"prefix {n} {cap} {dt}")


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 512, 64), (2, 2048, 128), (40, 1500, 32)])
def test_small_gradients_under_a_cap(Sq, Sk, D, dt):
    # dS of some 1e-5 and less is subnormal in fp16: rounded once, at its own size
    q, k, v, do = make(1, Sq, Sk, 2, 2, D, dt, seed=Sq)
    for kw in ({}, {"distance_slopes": torch.tensor([0.0625, 0.00390625], device=DEV)}):
        for cap in (2.0, 300.0):
            got, ref, names, _ = ts.run(q, k, v, do, softcap=cap, **dict(kw))
            oo.check(got, ref, names, f"{Sq} x {Sk}, {cap} {sorted(kw)}")
