"""flash_attention_v100_scored against the 64-bit oracle, element by element
within bounds from the arithmetic (tests/ops_oracle.py): every rule, type and
head dim, odd sizes, strides, masks that leave rows empty."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(B, Sq, Sk, H, Hkv, D, dt, seed=0, std=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * std).to(DT[dt]).to(DEV)  # noqa: E731
    return r(B, Sq, H, D), r(B, Sk, Hkv, D), r(B, Sk, Hkv, D), r(B, Sq, H, D)


def packed(B, S, lengths, pad=0):
    """ids 0, 1, .. of documents of these lengths (repeated to fill S), the last `pad` tokens -1."""
    out = torch.empty(B, S, dtype=torch.int32)
    for b in range(B):
        ids, n = [], b
        while len(ids) < S:
            ids += [n - b] * lengths[n % len(lengths)]
            n += 1
        out[b] = torch.tensor(ids[:S])
    if pad:
        out[:, S - pad:] = -1
    return out.to(DEV)


def run(q, k, v, do, train=True, **kw):
    """Kernel outputs and oracle for one call."""
    names = ["o", "lse"]
    slopes = kw.get("distance_slopes")
    if train:
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        if slopes is not None:
            kw["distance_slopes"] = slopes = slopes.detach().requires_grad_(True)
    o, lse = fa.flash_attention_v100_scored(q, k, v, return_softmax_lse=True, **kw)
    got = {"o": o.detach(), "lse": lse}
    if train:
        leaves = (q, k, v) + ((slopes,) if slopes is not None else ())
        grads = torch.autograd.grad(o, leaves, do)
        for n, t in zip(("dq", "dk", "dv", "dslopes"), grads):
            got[n] = t
            names.append(n)
    B, Sq = q.shape[:2]
    off = kw.get("query_offsets")
    off = 0 if off is None else off
    seen = oo.seen_mask(B, Sq, k.shape[1], kw.get("causal", False), kw.get("documents"), kw.get("key_documents"),
                        kw.get("prefix_lengths"), kw.get("key_lengths"), off, DEV)
    ref = oo.scored(q.detach(), k.detach(), v.detach(), do if train else None, kw.get("scale"),
                    kw.get("softcap") or 0.0, None if slopes is None else slopes.detach(), off, seen)
    return got, ref, names, seen


def slopes_for(H, B=None, seed=5):
    g = torch.Generator("cpu").manual_seed(seed)
    s = torch.exp2(-8.0 * torch.arange(1, H + 1) / H)
    s = s * (1 + 0.1 * torch.randn(H if B is None else (B, H), generator=g))
    return s.float().to(DEV)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rule", ["none", "cap", "slopes", "cap+slopes", "docs", "prefix"])
def test_rules_types_dims(rule, D, dt):
    B, S, H, Hkv = 2, 197, 4, 2
    print(f"case {rule} {D} {dt}", flush=True)
    q, k, v, do = make(B, S, S, H, Hkv, D, dt, seed=D)
    kw = {"causal": True}
    if "cap" in rule:
        kw["softcap"] = 3.0
    if "slopes" in rule:
        kw["distance_slopes"] = slopes_for(H)
    if rule == "docs":
        kw["documents"] = packed(B, S, [70, 3, 1, 55, 40])
    if rule == "prefix":
        kw["prefix_lengths"] = torch.tensor([0, 83], dtype=torch.int32, device=DEV)
    got, ref, names, _ = run(q, k, v, do, **kw)
    oo.check(got, ref, names, f"{rule} D={D} {dt}")


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 65), (33, 1), (64, 64), (65, 63), (128, 129), (130, 700), (700, 130)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(Sq, Sk, causal):
    q, k, v, do = make(1, Sq, Sk, 2, 1, 64, "bf16", seed=Sq + Sk)
    got, ref, names, _ = run(q, k, v, do, causal=causal, softcap=2.0, distance_slopes=slopes_for(2))
    oo.check(got, ref, names, f"{Sq} x {Sk}")


@pytest.mark.parametrize("D,dt", [(8, "fp16"), (20, "bf16"), (40, "fp16"), (80, "bf16"), (96, "fp16"), (100, "fp32"),
                                  (127, "bf16"), (3, "fp32")])
def test_head_dims_between(D, dt):
    q, k, v, do = make(2, 150, 150, 3, 3, D, dt, seed=D)
    got, ref, names, _ = run(q, k, v, do, causal=True, softcap=4.0)
    oo.check(got, ref, names, f"D={D} {dt}")


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_documents_unsorted_interleaved_and_padded(dt):
    # ids in any order, documents cut into pieces, ids far apart, padding inside and at the ends
    B, S = 3, 333
    g = torch.Generator("cpu").manual_seed(3)
    ids = torch.randint(0, 5, (B, S), generator=g, dtype=torch.int32) * 1000003
    ids[1] = torch.arange(S).flip(0) // 40
    ids[2] = -1
    ids[0, :70] = -5
    ids[1, 200:] = -1
    for causal in (True, False):
        q, k, v, do = make(B, S, S, 2, 2, 64, dt, seed=9)
        got, ref, names, seen = run(q, k, v, do, causal=causal, documents=ids.to(DEV))
        assert not seen[2].any()
        assert torch.equal(got["o"][2], torch.zeros_like(got["o"][2])) and (got["lse"][2] == -math.inf).all()
        for n in ("dq", "dk", "dv"):
            assert torch.equal(got[n][2], torch.zeros_like(got[n][2])), n
        oo.check(got, ref, names, f"unsorted {dt} causal={causal}")


def test_documents_long_sorted_and_cross():
    # many tiles, most of them skipped; more than 64 tiles of keys (two chunks of the walk)
    B, S = 1, 4500
    q, k, v, do = make(B, S, S, 2, 1, 32, "fp16", seed=4)
    got, ref, names, _ = run(q, k, v, do, causal=True, documents=packed(B, S, [900, 64, 1, 63, 130, 2000], pad=77))
    oo.check(got, ref, names, "long documents")
    q, k, v, do = make(2, 100, 260, 2, 1, 64, "bf16", seed=6)
    got, ref, names, _ = run(q, k, v, do, documents=packed(2, 100, [30, 11]), key_documents=packed(2, 260, [90, 70, 5]).long())
    oo.check(got, ref, names, "documents of queries and keys")


def test_one_dimensional_documents_are_shared():
    q, k, v, do = make(2, 140, 140, 2, 2, 64, "bf16", seed=8)
    d = packed(1, 140, [50, 31])[0]
    a = fa.flash_attention_v100_scored(q, k, v, documents=d)
    b = fa.flash_attention_v100_scored(q, k, v, documents=d.expand(2, 140).contiguous())
    assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_padding_values_reach_nothing(dt):
    # NaN and infinities in tokens of no document and behind the key lengths
    B, S = 2, 190
    q, k, v, do = make(B, S, S, 2, 1, 64, dt, seed=12)
    ids = packed(B, S, [60, 20])
    ids[0, 100:130] = -1
    ids[1, 150:] = -1
    bad = (ids < 0)
    clean = [t.clone() for t in (q, k, v, do)]
    for t, val in zip((q, k, v, do), (math.nan, math.inf, math.nan, math.nan)):
        t[bad] = val
    for t in clean:
        t[bad] = 0
    for kw in ({"causal": True}, {"softcap": 2.0}, {"distance_slopes": slopes_for(2)}):
        got, _, names, _ = run(q, k, v, do, documents=ids, **dict(kw))
        want, ref, _, _ = run(*clean, documents=ids, **dict(kw))
        for n in names:
            assert torch.equal(got[n], want[n]), (kw, n)
        oo.check(got, ref, names, str(list(kw)))
    lens = torch.tensor([100, 0], dtype=torch.int32, device=DEV)
    q, k, v, do = make(B, S, S, 2, 1, 64, dt, seed=13)
    k2, v2 = k.clone(), v.clone()
    for b in range(B):
        k2[b, int(lens[b]):] = math.nan
        v2[b, int(lens[b]):] = math.inf
    got, _, names, _ = run(q, k2, v2, do, causal=True, key_lengths=lens)
    want, ref, _, _ = run(q, k, v, do, causal=True, key_lengths=lens)
    for n in names:
        assert torch.equal(got[n], want[n]), n
    oo.check(want, ref, names, "key lengths")


def test_offsets_and_clamped_lengths():
    B, Sq, Sk = 4, 70, 200
    q, k, v, do = make(B, Sq, Sk, 2, 2, 64, "bf16", seed=14)
    off = torch.tensor([130, -40, 1 << 29, -(1 << 29)], dtype=torch.int32, device=DEV)
    got, ref, names, seen = run(q, k, v, do, causal=True, query_offsets=off)
    assert not seen[3].any() and not seen[1, :40].any() and seen[2].all()
    oo.check(got, ref, names, "offsets")
    # an int, and lengths past what exists or negative, count as all or nothing
    lens = torch.tensor([10 ** 6, -3, 5, 200], device=DEV)
    pre = torch.tensor([-7, 10 ** 8, 3, 100], dtype=torch.int32, device=DEV)
    got, _, names, _ = run(q, k, v, do, causal=True, query_offsets=17, key_lengths=lens, prefix_lengths=pre)
    seen = oo.seen_mask(B, Sq, Sk, True, None, None, pre.clamp(0, Sk), lens.clamp(0, Sk), 17, DEV)
    ref = oo.scored(q, k, v, do, None, 0.0, None, 17, seen)
    oo.check(got, ref, names, "clamped lengths")


def test_batch_slopes_and_shared_heads():
    B, S, H = 3, 160, 6
    q, k, v, do = make(B, S, S, H, 1, 64, "fp16", seed=15)
    got, ref, names, _ = run(q, k, v, do, distance_slopes=slopes_for(H, B), softcap=5.0)
    oo.check(got, ref, names, "slopes of each sequence, one KV head")


def test_strides_and_orders():
    B, S, H, D = 2, 170, 4, 64
    base = torch.randn(B, H, S, 3 * D, generator=torch.Generator("cpu").manual_seed(16)).to(torch.bfloat16).to(DEV)
    q, k, v = (base[..., i * D:(i + 1) * D].transpose(1, 2) for i in range(3))
    do = torch.randn(B, S, D, H, generator=torch.Generator("cpu").manual_seed(17)).to(torch.bfloat16).to(DEV).transpose(2, 3)
    got, ref, names, _ = run(q, k, v, do, causal=True, softcap=3.0)
    oo.check(got, ref, names, "packed projections, transposed gradient")
    # rows that no 16-byte load can read, and keys shared by the batch (stride 0)
    odd = torch.randn(B, S, H, D + 1, generator=torch.Generator("cpu").manual_seed(18)).to(torch.bfloat16).to(DEV)[..., 1:]
    k1 = k[:1].expand(B, S, H, D)
    got, ref, names, _ = run(odd, k1, v, do, causal=True)
    oo.check(got, ref, names, "odd rows, shared keys")


def test_same_as_the_dense_attention():
    # no rule: the library's causal attention, within the bounds of both
    q, k, v, do = make(2, 300, 300, 4, 2, 128, "bf16", seed=19)
    got, ref, names, _ = run(q, k, v, do, causal=True)
    o = fa.flash_attention_v100(q, k, v, causal=True)
    oo.check({"o": o}, ref, ["o"], "dense")
    oo.check(got, ref, names, "scored")


@pytest.mark.parametrize("Sq", [1, 2, 5, 16])
@pytest.mark.parametrize("dt,D", [("bf16", 128), ("fp16", 64), ("fp32", 64), ("fp32", 128), ("bf16", 32), ("fp16", 72)])
def test_tokens_over_a_cache(dt, D, Sq):
    B, Sk, H, Hkv = 5, 1000, 8, 2
    q, k, v, _ = make(B, Sq, Sk, H, Hkv, D, dt, seed=20 + Sq)
    lens = torch.tensor([1000, 513, 64, max(1, Sq - 1), 0], dtype=torch.int32, device=DEV)
    for b in range(B):  # an unfilled cache holds anything
        k[b, int(lens[b]):] = math.nan
        v[b, int(lens[b]):] = math.nan
    kz, vz = torch.nan_to_num(k), torch.nan_to_num(v)
    for kw in ({}, {"softcap": 4.0}, {"distance_slopes": slopes_for(H)}):
        got = dict(zip(("o", "lse"), fa.flash_attention_v100_scored(
            q, k, v, causal=True, key_lengths=lens, query_offsets=lens - Sq, return_softmax_lse=True, **kw)))
        seen = oo.seen_mask(B, Sq, Sk, True, None, None, None, lens, lens - Sq, DEV)
        ref = oo.scored(q, kz, vz, None, None, kw.get("softcap", 0.0), kw.get("distance_slopes"), lens - Sq, seen)
        oo.check(got, ref, ["o", "lse"], f"{dt} D={D} Sq={Sq} {list(kw)}")


def test_token_gradients():
    # few rows take another forward kernel: its LSE serves the backward
    q, k, v, do = make(3, 2, 400, 4, 2, 64, "bf16", seed=30)
    lens = torch.tensor([400, 100, 1], dtype=torch.int32, device=DEV)
    got, ref, names, _ = run(q, k, v, do, causal=True, key_lengths=lens, query_offsets=lens - 2,
                             distance_slopes=slopes_for(4))
    oo.check(got, ref, names, "two tokens")


def test_empty_tensors():
    for B, Sq, Sk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q, k, v, do = make(B, Sq, Sk, 2, 2, 64, "bf16")
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
        s = slopes_for(2).requires_grad_(True)
        o, lse = fa.flash_attention_v100_scored(q, k, v, causal=True, distance_slopes=s, return_softmax_lse=True)
        assert o.shape == q.shape and not o.any() and (lse == -math.inf).all()
        for g in torch.autograd.grad(o, (q, k, v, s), do):
            assert not g.any()


def test_large_scores_and_infinities():
    # scores far past the cap: tanh at its ends; a NaN query row stays in its row
    q, k, v, do = make(1, 130, 130, 2, 2, 64, "bf16", seed=31, std=30.0)
    got, ref, names, _ = run(q, k, v, do, causal=True, softcap=10.0)
    oo.check(got, ref, ["o", "lse", "dv"], "saturated cap")
    for n in names:
        assert torch.isfinite(got[n]).all(), n
    q, k, v, do = make(1, 130, 130, 2, 2, 64, "bf16", seed=32)
    want = fa.flash_attention_v100_scored(q, k, v, causal=True, softcap=10.0)
    q[0, 77, 1] = math.nan
    o = fa.flash_attention_v100_scored(q, k, v, causal=True, softcap=10.0)
    assert torch.isnan(o[0, 77, 1]).all()
    o[0, 77, 1] = want[0, 77, 1]
    assert torch.equal(o, want)


def test_gradients_against_differences():
    # float32 against central differences of the 64-bit definition
    B, S, H, D = 1, 37, 2, 16
    q, k, v, do = make(B, S, S, H, 1, D, "fp32", seed=33)
    sl = slopes_for(H)
    kw = {"causal": True, "softcap": 2.5, "documents": packed(B, S, [20, 9])}
    got, _, _, seen = run(q, k, v, do, distance_slopes=sl, **kw)

    def loss(q, k, v, s):
        x = oo._heads(q, H) @ oo._heads(k, H).transpose(-1, -2) * D ** -0.5
        x = 2.5 * torch.tanh(x / 2.5)
        i = torch.arange(S, device=DEV)
        x = x - s.double().view(1, H, 1, 1) * (i[:, None] - i[None, :]).abs()
        p = torch.softmax(x.masked_fill(~seen.unsqueeze(1), -math.inf), -1)
        return ((p @ oo._heads(v, H)).transpose(1, 2) * do.double()).sum()

    leaves = [t.double() for t in (q, k, v, sl)]
    g = torch.Generator("cpu").manual_seed(34)
    for n, name in enumerate(("dq", "dk", "dv", "dslopes")):
        step = torch.randn(leaves[n].shape, generator=g, dtype=torch.float64).to(DEV)
        h = 1e-5
        plus, minus = [list(leaves) for _ in range(2)]
        plus[n], minus[n] = leaves[n] + h * step, leaves[n] - h * step
        num = ((loss(*plus) - loss(*minus)) / (2 * h)).item()
        ana = (got[name].double() * step).sum().item()
        # the sums of |gradient||step| in float32 roundings along some tens of steps, and h^2 of the difference
        tol = 2.0 ** -18 * (got[name].double().abs() * step.abs()).sum().item() + 1e-7 * abs(num) + 1e-7
        print(f"{name}: {ana:.8f} against {num:.8f}, tolerance {tol:.2e}", flush=True)
        assert abs(num - ana) <= tol


@pytest.mark.parametrize("Sq", [1, 20, 200])
def test_without_lse(Sq):
    q, k, v, _ = make(2, Sq, 200, 4, 2, 64, "bf16", seed=12)
    for kw in (dict(causal=True), dict(softcap=9.0, documents=torch.zeros(Sq, dtype=torch.int32, device=DEV),
                                       key_documents=torch.zeros(200, dtype=torch.int32, device=DEV))):
        o, lse = fa.flash_attention_v100_scored(q, k, v, return_softmax_lse=True, **kw)
        assert torch.equal(fa.flash_attention_v100_scored(q, k, v, **kw), o) and lse.shape == (2, 4, Sq)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rule", ["none", "cap", "slopes", "cap+slopes", "docs", "prefix", "all keys"])
def test_rules_on_larger_grids(rule, D, dt):
    # 600 blocks of queries and of keys: one group of waves each, no parts
    B, S, H, Hkv = 5, 500, 30, 30
    q, k, v, do = make(B, S, S, H, Hkv, D, dt, seed=D)
    kw = dict(causal=rule != "all keys")
    if "cap" in rule:
        kw["softcap"] = 5.0
    if "slopes" in rule:
        kw["distance_slopes"] = slopes_for(H)
    if rule == "docs":
        kw["documents"] = packed(B, S, [97, 230, 14], pad=9)
    if rule == "prefix":
        kw["prefix_lengths"] = torch.tensor([0, 60, 129, 500, 3], device=DEV, dtype=torch.int32)
        kw["key_lengths"] = torch.tensor([500, 490, 200, 500, 1], device=DEV, dtype=torch.int32)
    got, ref, names, _ = run(q, k, v, do, **kw)
    oo.check(got, ref, names, f"{rule} {dt} {D}")


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,Sq,Sk,H,Hkv,D", [(1, 100, 900, 8, 2, 128), (2, 33, 400, 6, 1, 64), (1, 300, 1300, 4, 4, 32),
                                             (40, 20, 90, 6, 2, 64)])
def test_chunks_over_a_cache(B, Sq, Sk, H, Hkv, D, dt):
    # many queries at the end of longer caches, filled to different lengths
    q, k, v, _ = make(B, Sq, Sk, H, Hkv, D, dt, seed=Sq)
    lens = torch.randint(Sq // 2, Sk + 1, (B,), generator=torch.Generator("cpu").manual_seed(Sq)).to(DEV)
    for kw in (dict(causal=True), dict(), dict(causal=True, softcap=7.0, distance_slopes=slopes_for(H))):
        got, ref, names, _ = run(q, k, v, None, False, key_lengths=lens, query_offsets=lens - Sq, **kw)
        oo.check(got, ref, names, f"{dt} {sorted(kw)}")
