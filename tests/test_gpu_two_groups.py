"""flash_attention_v100_scored on grids of fewer workgroups than CUs over 512 keys and
more, whose blocks have two groups of waves: every rule, type and compiled head dim,
odd sizes, against the 64-bit oracle; few rows in one part and in several."""
import pytest
import torch

import ops_oracle as oo
from test_gpu_scored import make, packed, run, slopes_for

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
@pytest.mark.parametrize("rule", ["none", "all keys", "cap", "slopes", "cap+slopes", "docs", "prefix", "lengths"])
def test_rules(rule, D, dt):
    B, S, H, Hkv = 2, 587, 2, 1
    q, k, v, do = make(B, S, S, H, Hkv, D, dt, seed=D)
    kw = {"causal": rule != "all keys"}
    if "cap" in rule:
        kw["softcap"] = 3.0
    if "slopes" in rule:
        kw["distance_slopes"] = slopes_for(H)
    if rule == "docs":
        kw["documents"] = packed(B, S, [130, 3, 1, 95, 40], pad=13)
    if rule == "prefix":
        kw["prefix_lengths"] = torch.tensor([0, 303], dtype=torch.int32, device=DEV)
    if rule == "lengths":
        kw.update(key_lengths=torch.tensor([1, 530], dtype=torch.int32, device=DEV), query_offsets=-20)
    got, ref, names, _ = run(q, k, v, do, **kw)
    oo.check(got, ref, names, f"{rule} D={D} {dt}")


@pytest.mark.parametrize("Sq,Sk", [(1, 512), (130, 513), (700, 512), (33, 1025)])
def test_lengths(Sq, Sk):
    q, k, v, do = make(1, Sq, Sk, 2, 2, 64, "fp16", seed=Sq)
    for causal in (True, False):
        got, ref, names, _ = run(q, k, v, do, causal=causal, softcap=2.0, distance_slopes=slopes_for(2))
        oo.check(got, ref, names, f"{Sq} x {Sk}")


@pytest.mark.parametrize("Sk", [64, 960, 961, 1023, 1024, 1025, 1537])
@pytest.mark.parametrize("B,Sq", [(1, 1), (3, 5), (64, 15)])
def test_parts_of_few_rows(B, Sq, Sk):
    # one part up to 960 keys; then parts of 512, or of what fills the device once
    q, k, v, _ = make(B, Sq, Sk, 8, 2, 64, "bf16", seed=Sk)
    got, ref, names, _ = run(q, k, v, None, False, causal=True, query_offsets=Sk - Sq, softcap=5.0)
    oo.check(got, ref, names, f"{B} x {Sq} x {Sk}")
