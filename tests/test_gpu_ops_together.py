"""The operators around attention as a program uses them: one after the other in
training and in serving, in the layer, in captured graphs, on other streams,
over caches past 32-bit offsets, and what they refuse."""
import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo
from flash_attention_v100 import _ops
from test_gpu_scored import DT, make, packed, run, slopes_for

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---------------------------------------------------------------------------
# one after the other
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_training_step(dt):
    # rotary positions that start again with each document, capped scores, slopes
    # and documents; gradients through both operators
    B, S, H, Hkv, D = 2, 333, 4, 2, 64
    q, k, v, do = make(B, S, S, H, Hkv, D, dt, seed=3)
    docs = packed(B, S, [100, 37, 64, 1], pad=11)
    first = (docs[:, :, None] == docs[:, None, :]).int().argmax(-1)
    pos = torch.arange(S, device=DEV, dtype=torch.int32) - first.int()
    table = fa.rotary_table_v100(S, D)
    slopes = slopes_for(H)
    kw = dict(causal=True, softcap=20.0, documents=docs)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, slopes)]
    rq, rk = fa.rotary_embedding_v100(leaves[0], leaves[1], table, pos)
    o, lse = fa.flash_attention_v100_scored(rq, rk, leaves[2], distance_slopes=leaves[3], return_softmax_lse=True, **kw)
    grads = torch.autograd.grad(o, leaves, do)
    # the attention on the rotated inputs, then its gradients turned back
    got, ref, names, _ = run(rq.detach(), rk.detach(), v, do, distance_slopes=slopes, **kw)
    oo.check(got, ref, names, dt)
    assert torch.equal(o, got["o"]) and torch.equal(lse, got["lse"])
    assert torch.equal(grads[2], got["dv"]) and torch.equal(grads[3], got["dslopes"])
    w, mul = oo.frequencies(D)
    for g, d, n in ((grads[0], got["dq"], "dq"), (grads[1], got["dk"], "dk")):
        val, bound = oo.rotate(d, pos, w, mul, False, inverse=True)
        oo.check({n: g}, {n: (val, bound)}, [n], "turned back")


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_serving_steps(dt):
    # a prompt read once, then tokens of 5 sequences (one slot free) that go on from
    # it, rotated in place and written to the sequences' own caches
    B, P, cap, H, Hkv, D = 5, 150, 24, 8, 2, 64
    g = torch.Generator("cpu").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(DT[dt]).to(DEV)  # noqa: E731
    table = fa.rotary_table_v100(P + cap, D)
    pq, pk, pv = r(1, P, H, D), r(1, P, Hkv, D), r(1, P, Hkv, D)
    fa.rotary_embedding_v100(pq, pk, table, inplace=True)
    o = fa.flash_attention_v100_scored(pq, pk, pv, causal=True, softcap=30.0)
    ref = oo.scored(pq, pk, pv, softcap=30.0, seen=oo.seen_mask(1, P, P, True, device=DEV))
    oo.check({"o": o}, ref, ["o"], "prompt")
    kc, vc = torch.full((B, cap, Hkv, D), float("nan"), device=DEV, dtype=DT[dt]), r(B, cap, Hkv, D)
    live = torch.tensor([1, 1, 0, 1, 1], device=DEV)
    lens = torch.zeros(B, dtype=torch.int64, device=DEV)
    for step in (1, 3, 1, 2):
        q, k, v = r(B, step, H, D), r(B, step, Hkv, D), r(B, step, Hkv, D)
        pos = torch.where(live.bool()[:, None], P + lens[:, None] + torch.arange(step, device=DEV), -1)
        fa.rotary_embedding_v100(q, k, table, pos, inplace=True)
        for b in range(B):
            if live[b]:
                n = int(lens[b])
                kc[b, n:n + step], vc[b, n:n + step] = k[b], v[b]
        lens = lens + step * live
        o, lse = fa.flash_attention_v100_shared_prefix(q, pk[0], pv[0], kc, vc, lens, softcap=30.0,
                                                       return_softmax_lse=True)
        own = lens.view(B, 1) - step + torch.arange(step, device=DEV)
        j = torch.arange(P + cap, device=DEV) - P
        seen = (j <= own[..., None]) & (own[..., None] >= 0)
        ref = oo.scored(q, torch.cat([pk.expand(B, -1, -1, -1), kc.nan_to_num()], 1),
                        torch.cat([pv.expand(B, -1, -1, -1), vc], 1), softcap=30.0, seen=seen)
        oo.check({"o": o, "lse": lse}, ref, ["o", "lse"], f"step of {step}")
        assert torch.equal(o[2], torch.zeros_like(o[2])) and (lse[2] == -float("inf")).all()
        # the same tokens over one cache that holds prompt and own keys
        whole = torch.cat([pk.expand(B, -1, -1, -1), kc], 1), torch.cat([pv.expand(B, -1, -1, -1), vc], 1)
        seq = live.bool()
        o2 = fa.flash_attention_v100_scored(q[seq], whole[0][seq], whole[1][seq], causal=True, softcap=30.0,
                                            key_lengths=(P + lens)[seq], query_offsets=(P + lens - step)[seq])
        oo.check({"o": o2}, {"o": tuple(t[seq] for t in ref["o"])}, ["o"], "one cache")


# ---------------------------------------------------------------------------
# the layer
def _plain_layer(m, x, positions, documents, pad, causal):
    """The layer in 64 bits on the CPU, differentiable."""
    P = {n: p.detach().double().cpu().requires_grad_(True) for n, p in m.named_parameters()}
    x = x.detach().double().cpu()
    B, S, E = x.shape
    H, D = m.num_heads, m.head_dim
    lin = lambda n, t: t @ P[n + ".weight"].T + P[n + ".bias"]  # noqa: E731
    q, k, v = (lin(n, x).view(B, S, H, D) for n in ("q_proj", "k_proj", "v_proj"))
    R = m.rotary_dim
    if R:
        w, mul = oo.frequencies(R, m.rotary_base, **{{"original_positions": "original"}.get(a, a): b
                                                      for a, b in m.rotary_scaling.items()})
        ang = positions.cpu().double().expand(B, S).view(B, S, 1, 1) * w
        c, s = torch.cos(ang) * mul, torch.sin(ang) * mul

        def turn(t):
            a, b = (t[..., 0:R:2], t[..., 1:R:2]) if m.rotary_interleaved else (t[..., :R // 2], t[..., R // 2:R])
            y, z = a * c - b * s, b * c + a * s
            y = torch.stack((y, z), -1).flatten(-2) if m.rotary_interleaved else torch.cat((y, z), -1)
            return torch.cat((y, t[..., R:]), -1)
        q, k = turn(q), turn(k)
    sc = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    if m.softcap:
        sc = m.softcap * torch.tanh(sc / m.softcap)
    d = (torch.arange(S).view(S, 1) - torch.arange(S)).abs().double()
    if m.distance_slopes is not None:
        sc = sc - P["distance_slopes"].view(H, 1, 1) * d
    docs = documents.cpu() if documents is not None else None
    kd = (torch.zeros(B, S) if docs is None else docs.expand(B, S)).masked_fill(
        pad.cpu() if pad is not None else torch.zeros(B, S, dtype=torch.bool), -1)
    seen = oo.seen_mask(B, S, S, causal, torch.zeros(B, S) if docs is None else docs, kd)
    sc = sc.masked_fill(~seen.unsqueeze(1), -float("inf"))
    p = torch.nan_to_num(torch.softmax(sc, -1))
    o = torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, S, E)
    return lin("out_proj", o), P


@pytest.mark.parametrize("case", [
    dict(rotary_dim=32), dict(rotary_dim=16, rotary_interleaved=True, pos=True),
    dict(softcap=8.0, pad=True), dict(distance_bias=True, causal=True),
    dict(rotary_dim=32, rotary_scaling=dict(scaling="ramp", factor=4.0, original_positions=64), softcap=8.0,
         distance_bias=True, docs=True, pos=True, pad=True, causal=True)], ids=lambda c: "+".join(c))
def test_layer(case):
    # fp32.  Scores of at most 6 or so in magnitude sum 32 products (2 w each), the
    # cap adds 8 x 2^-21: a probability is off by 2 x (6 x 64 w + 2^-18) = 5e-5 of
    # itself, twice that in a gradient, and the projections add 256 w of their size
    torch.manual_seed(0)
    B, S, E, H = 2, 96, 128, 4
    opts = {n: case[n] for n in ("rotary_dim", "rotary_interleaved", "rotary_scaling", "softcap", "distance_bias") if n in case}
    m = fa.EnhancedMultiHeadAttention(E, H, **opts).to(DEV)
    x = torch.randn(B, S, E, device=DEV)
    docs = packed(B, S, [40, 17, 30]) if case.get("docs") else None
    pos = torch.randint(0, 300, (B, S), device=DEV) if case.get("pos") else torch.arange(S, device=DEV)
    pad = None
    if case.get("pad"):
        pad = torch.zeros(B, S, dtype=torch.bool, device=DEV)
        pad[1, 70:] = True
    causal = case.get("causal", False)
    out, _ = m(x, key_padding_mask=pad, is_causal=causal, documents=docs, positions=pos if case.get("pos") else None)
    do = torch.randn_like(out)
    out.backward(do)
    ref, P = _plain_layer(m, x, pos, docs, pad, causal)
    ref.backward(do.double().cpu())
    err = (out.detach().cpu().double() - ref.detach()).abs().max().item()
    print("out", err, ref.abs().max().item(), flush=True)
    assert err <= 2e-4 * ref.abs().max().item()
    big = max(P[n].grad.abs().max().item() for n in P)
    for n, p in m.named_parameters():
        e, t = (p.grad.cpu().double() - P[n].grad).abs().max().item(), P[n].grad.abs().max().item()
        print(n, e, t, flush=True)
        assert e <= max(2e-4 * t, 1e-5 * big), n


def test_layer_16_bit_masks_and_capture():
    torch.manual_seed(0)
    m = fa.EnhancedMultiHeadAttention(128, 4, rotary_dim=32, distance_bias=True).to(DEV).to(torch.bfloat16).eval()
    x = torch.randn(2, 50, 128, device=DEV, dtype=torch.bfloat16)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="once before it is captured"):
        with torch.cuda.graph(g):
            m(x)
    torch.cuda.synchronize()
    with torch.no_grad():
        want = m(x)[0]
        # padding as a mask and as documents
        pad = torch.zeros(2, 50, dtype=torch.bool, device=DEV)
        pad[0, 41:] = True
        a = m(x, key_padding_mask=pad)[0]
        b = m(x, documents=torch.where(pad, -1, 0))[0]
        assert torch.equal(a[~pad], b[~pad])
        with pytest.raises(ValueError, match="attn_mask"):
            m(x, attn_mask=torch.zeros(50, 50, dtype=torch.bool, device=DEV))
        with pytest.raises(ValueError, match="max_positions"):
            fa.EnhancedMultiHeadAttention(128, 4, rotary_dim=32, max_positions=49).to(DEV)(x.float())
    assert torch.isfinite(want.float()).all()


# ---------------------------------------------------------------------------
# captured graphs
def _scored_calls():
    docs = packed(2, 300, [90, 45, 64], pad=7)
    lens = torch.tensor([300, 170], device=DEV, dtype=torch.int32)
    return {
        "cap": (dict(causal=True, softcap=10.0), (2, 300, 300, 4, 2, 64, "bf16")),
        "slopes+docs": (dict(causal=True, documents=docs), (2, 300, 300, 4, 4, 64, "fp16")),
        "prefix": (dict(causal=True, prefix_lengths=lens // 2, key_lengths=lens), (2, 300, 300, 2, 1, 80, "fp32")),
        "parts": (dict(causal=True), (1, 2048, 2048, 4, 1, 64, "bf16")),
    }


@pytest.mark.parametrize("name", ["cap", "slopes+docs", "prefix", "parts"])
def test_training_graph(name):
    kw, shape = _scored_calls()[name]
    q, k, v, do = make(*shape, seed=2)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    if "slopes" in name:
        leaves.append(slopes_for(shape[3]).requires_grad_(True))
        kw["distance_slopes"] = leaves[3]

    def step():
        o = fa.flash_attention_v100_scored(q, k, v, **kw)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, do))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for n, t in enumerate((q, k, v, do)):
                t.copy_(make(*shape, seed=10 + i)[n])
        want = [t.clone() for t in step()]
        junk = torch.randn(1 << 20, device=DEV).sum()
        g.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(junk)
        for a, b in zip(out, want):
            assert torch.equal(a, b), (name, i)


def test_capture_refuses_inputs_of_a_living_graph(monkeypatch):
    # a captured backward of leaves that an eager graph of another stream holds would
    # end the process: refused.  The capture is pretended, no graph is recorded
    q, k, v, do = make(1, 40, 40, 2, 2, 32, "bf16")
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    table = fa.rotary_table_v100(40, 32)
    calls = (lambda: fa.flash_attention_v100_scored(q, k, v), lambda: fa.rotary_embedding_v100(q, k, table))
    for call in calls:
        alive = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            with torch.cuda.stream(side):
                with pytest.raises(RuntimeError, match="still alive"):
                    call()
                del alive
                call()
                moved = q * 1  # made here: its gradient stays on this stream
                fa.flash_attention_v100_scored(moved, k, v)
            with pytest.raises(RuntimeError, match="still alive"):
                fa.flash_attention_v100_scored(moved, k, v)
            with torch.no_grad():
                call()
        torch.cuda.synchronize()
        del moved


def test_serving_graphs_that_share_a_pool():
    # two graphs (other batch sizes) with one memory pool, replayed in turn as their
    # lengths and positions grow in place
    H, Hkv, D, P, cap = 8, 2, 128, 700, 64
    g0 = torch.Generator("cpu").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g0).to(torch.bfloat16).to(DEV)  # noqa: E731
    kp, vp = r(P, Hkv, D), r(P, Hkv, D)
    table = fa.rotary_table_v100(P + cap, D)
    pool, steps = None, []
    for B in (3, 40):
        t = dict(q=r(B, 1, H, D), k=r(B, cap, Hkv, D), v=r(B, cap, Hkv, D),
                 lens=torch.randint(0, 20, (B,), generator=g0).to(torch.int32).to(DEV))

        def step(t=t):
            q = fa.rotary_embedding_v100(t["q"], None, table, P + t["lens"].view(-1, 1) - 1)
            o = fa.flash_attention_v100_shared_prefix(q, kp, vp, t["k"], t["v"], t["lens"], softcap=25.0)
            c = fa.flash_attention_v100_scored(q, t["k"], t["v"], causal=True, key_lengths=t["lens"],
                                               query_offsets=t["lens"] - 1)
            return o, c
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            out = step()
        pool = g.pool()
        steps.append((g, step, t, out))
    for _ in range(4):
        for g, step, t, out in steps:
            t["lens"].add_(7)
            t["q"].copy_(torch.randn(t["q"].shape, generator=g0).to(torch.bfloat16))
            want = [x.clone() for x in step()]
            junk = torch.randn(1 << 20, device=DEV).sum()
            g.replay()
            torch.cuda.synchronize()
            assert torch.isfinite(junk)
            for a, b in zip(out, want):
                assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# streams, repeated calls, far offsets
def test_other_streams_and_repeated_calls():
    shape = (1, 1500, 1500, 4, 2, 64, "bf16")
    q, k, v, do = make(*shape, seed=6)
    docs, slopes, table = packed(1, 1500, [400, 77]), slopes_for(4), fa.rotary_table_v100(1500, 64)

    def work():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, slopes)]
        rq, rk = fa.rotary_embedding_v100(leaves[0], leaves[1], table)
        o = fa.flash_attention_v100_scored(rq, rk, leaves[2], causal=True, documents=docs, distance_slopes=leaves[3])
        g = torch.autograd.grad(o, leaves, do)
        p = fa.flash_attention_v100_shared_prefix(q[:, :3], k[0], v[0], k[:, :40], v[:, :40])
        return [o.detach(), p, *g]

    want = work()
    again = work()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(work())
    torch.cuda.synchronize()
    for got in [again] + outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)  # no atomics: the same bits on any stream


def test_offsets_past_32_bits():
    # a cache of 2.5e9 elements: as 3 sequences of 200000 keys, and as one prefix
    B, S, Hkv, D = 3, 204800, 32, 128
    k = torch.empty(B, S, Hkv, D, device=DEV, dtype=torch.bfloat16).normal_()
    v = torch.empty_like(k).normal_()
    q = torch.randn(B, 1, Hkv, D, device=DEV).to(torch.bfloat16)
    lens = torch.tensor([3, 100000, S - 1], device=DEV)
    o, lse = fa.flash_attention_v100_scored(q, k, v, causal=True, key_lengths=lens, query_offsets=lens - 1,
                                            return_softmax_lse=True)
    for b in (1, 2):
        for h in (0, 31):
            kk, vv = (t[b:b + 1, :, h:h + 1].contiguous() for t in (k, v))
            ref = oo.scored(q[b:b + 1, :, h:h + 1], kk, vv, seen=oo.seen_mask(1, 1, S, lens=lens[b:b + 1], device=DEV))
            oo.check({"o": o[b:b + 1, :, h:h + 1], "lse": lse[b:b + 1, h:h + 1]}, ref, ["o", "lse"], f"cache {b} {h}")
    kp, vp = k.view(B * S, Hkv, D), v.view(B * S, Hkv, D)
    own = torch.randn(2, 4, Hkv, D, device=DEV).to(torch.bfloat16)
    q2 = q[:2]
    o, lse = fa.flash_attention_v100_shared_prefix(q2, kp, vp, own, own, return_softmax_lse=True)
    for h in (0, 31):
        kk = torch.cat([kp[:, h], own[1, :, h]]).view(1, -1, 1, D)
        vv = torch.cat([vp[:, h], own[1, :, h]]).view(1, -1, 1, D)
        ref = oo.scored(q2[1:, :, h:h + 1], kk, vv, seen=torch.ones(1, 1, kk.shape[1], dtype=torch.bool, device=DEV))
        oo.check({"o": o[1:, :, h:h + 1], "lse": lse[1:, h:h + 1]}, ref, ["o", "lse"], f"prefix {h}")


def test_rows_far_apart():
    # rows 2^20 elements apart: offsets of 2^32 elements inside one sequence
    S, H, D, row = 4200, 2, 64, 1 << 20
    buf = torch.empty(S * row, device=DEV, dtype=torch.bfloat16)
    views, plain = [], []
    for n in range(4):
        x = torch.randn(1, S, H, D, device=DEV).to(torch.bfloat16)
        t = buf.as_strided((1, S, H, D), (S * row, row, D, 1), n * H * D)
        t.copy_(x)
        views.append(t)
        plain.append(x)
    outs = []
    for q, k, v, do in (views, plain):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = fa.flash_attention_v100_scored(*leaves, causal=True, softcap=20.0)
        outs.append([o.detach(), *torch.autograd.grad(o, leaves, do)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    table = fa.rotary_table_v100(S, D)
    a, b = (fa.rotary_embedding_v100(t[0], t[1], table) for t in (views, plain))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_64_bit_lengths_and_ids_keep_their_meaning():
    q, k, v, _ = make(2, 70, 70, 2, 2, 32, "fp16", seed=8)
    big = torch.tensor([1 << 33, 50], device=DEV)
    a = fa.flash_attention_v100_scored(q, k, v, key_lengths=big)
    b = fa.flash_attention_v100_scored(q, k, v, key_lengths=torch.tensor([70, 50], device=DEV))
    assert torch.equal(a, b)
    a = fa.flash_attention_v100_scored(q, k, v, causal=True, query_offsets=torch.tensor([1 << 33, -(1 << 33)], device=DEV))
    assert torch.equal(a[0], fa.flash_attention_v100_scored(q, k, v)[0]) and torch.equal(a[1], torch.zeros_like(a[1]))
    ids = torch.zeros(70, dtype=torch.int64, device=DEV)
    ids[40:] = 1 << 32
    pad = torch.zeros(70, dtype=torch.int32, device=DEV)
    pad[40:] = -1
    assert torch.equal(fa.flash_attention_v100_scored(q, k, v, documents=ids),
                       fa.flash_attention_v100_scored(q, k, v, documents=pad))


# ---------------------------------------------------------------------------
# refusals that need tensors of the device (none reaches a kernel)
def test_scored_refusals():
    q, k, v, _ = make(2, 20, 30, 4, 2, 32, "fp16")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=1e-9),
               dict(distance_slopes=f32(3)), dict(distance_slopes=f32(4).half()), dict(distance_slopes=f32(4).cpu()),
               dict(distance_slopes=f32(2, 4, 1)), dict(documents=i32(2, 20)), dict(key_documents=i32(2, 30)),
               dict(documents=i32(2, 20), key_documents=i32(2, 20)), dict(documents=f32(20), key_documents=i32(30)),
               dict(documents=i32(20).cpu(), key_documents=i32(30)), dict(prefix_lengths=i32(2)),
               dict(causal=True, prefix_lengths=i32(3)), dict(key_lengths=i32(2, 1)), dict(key_lengths=f32(2)),
               dict(query_offsets=i32(3)), dict(query_offsets=1 << 31)):
        with pytest.raises(ValueError):
            fa.flash_attention_v100_scored(q, k, v, **kw)
    for kw in (dict(distance_slopes=[0.0] * 4), dict(documents=[0] * 20), dict(key_lengths=3)):
        with pytest.raises(TypeError):
            fa.flash_attention_v100_scored(q, k, v, **kw)
    with pytest.raises(NotImplementedError):
        fa.flash_attention_v100_scored(*(torch.zeros(1, 4, 2, 136, device=DEV).half() for _ in range(3)))
    with pytest.raises(ValueError):
        fa.flash_attention_v100_shared_prefix(q, k[0, :, :1], v[0], k, v)
    with pytest.raises(ValueError):
        fa.flash_attention_v100_shared_prefix(q, k[0].float(), v[0].float(), k, v)
    with pytest.raises(TypeError):
        fa.flash_attention_v100_shared_prefix(q, k[0], None, k, v)


def test_rotary_refusals():
    q, k, _, _ = make(2, 20, 20, 4, 2, 32, "fp16")
    table = fa.rotary_table_v100(20, 32)
    for args, kw in (((q, k, table.half()), {}), ((q, k, table[0]), {}), ((q, k, table[:, :3]), {}), ((q, k, table.cpu()), {}),
                     ((q, k, fa.rotary_table_v100(20, 64)), {}), ((q, k[:, :5], table), {}), ((q, k.float(), table), {}),
                     ((q, k, table, torch.zeros(20, device=DEV)), {}),
                     ((q, k, table, torch.zeros(19, dtype=torch.int32, device=DEV)), {}),
                     ((q, k, table, torch.zeros(20, dtype=torch.int32)), {}),
                     ((q, k, table.clone().requires_grad_(True)), {}),
                     ((q, q, table), dict(inplace=True)), ((q, q[:, :, 1:3], table), dict(inplace=True)),
                     ((q.expand(2, 20, 4, 32)[:, :1].expand(2, 20, 4, 32), k, table), dict(inplace=True)),
                     ((q.detach().requires_grad_(True), k, table), dict(inplace=True))):
        with pytest.raises(ValueError):
            fa.rotary_embedding_v100(*args, **kw)
    # heads of one packed tensor are fine, and their gradients' version moves on
    x = torch.randn(2, 20, 6, 32, device=DEV).half()
    want = fa.rotary_embedding_v100(x[:, :, :4], x[:, :, 4:], table)
    y = x.clone()
    n = y._version
    fa.rotary_embedding_v100(y[:, :, :4], y[:, :, 4:], table, inplace=True)
    assert torch.equal(y[:, :, :4], want[0]) and torch.equal(y[:, :, 4:], want[1]) and y._version > n
    assert _ops.MAX_HEAD_DIM == 128


# ---------------------------------------------------------------------------
# the C ABI itself, as a program without the Python entry points calls it
def test_c_abi():
    import ctypes

    lib, stream = _ops.load(), torch.cuda.current_stream().cuda_stream
    B, S, H, Hkv, D = 2, 300, 4, 2, 64
    q, k, v, do = make(B, S, S, H, Hkv, D, "bf16", seed=9)
    docs, slopes = packed(B, S, [100, 70], pad=5), slopes_for(H)
    lens = torch.tensor([300, 211], device=DEV, dtype=torch.int32)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, slopes)]
    o, lse = fa.flash_attention_v100_scored(*leaves[:3], causal=True, softcap=11.0, distance_slopes=leaves[3], documents=docs,
                                            key_lengths=lens, return_softmax_lse=True)
    want = [o.detach(), lse, *torch.autograd.grad(o, leaves, do)]
    out = [torch.full_like(t, float("nan")) for t in want]

    a = _ops.ScoredArgs()
    for n, t in zip(("q", "k", "v", "dout", "o", "dq", "dk", "dv"), (q, k, v, do, out[0], *out[2:5])):
        setattr(a, n, t.data_ptr())
        getattr(a, ("do" if n == "dout" else n) + "_stride")[:] = t.stride()
    a.lse, a.slopes, a.dslopes, a.key_lengths = out[1].data_ptr(), slopes.data_ptr(), out[5].data_ptr(), lens.data_ptr()
    a.q_documents = a.k_documents = docs.data_ptr()
    a.q_documents_stride = a.k_documents_stride = S
    a.batch, a.seqlen_q, a.seqlen_k, a.num_heads, a.num_heads_kv, a.head_dim, a.dtype, a.causal = B, S, S, H, Hkv, D, 1, 1
    a.scale, a.softcap = D ** -0.5, 11.0
    for size, call in ((lib.fa_scored_fwd_workspace_size, lib.fa_scored_fwd),
                       (lib.fa_scored_bwd_workspace_size, lib.fa_scored_bwd)):
        n = size(ctypes.byref(a))
        ws = torch.full((n + 256,), 255, device=DEV, dtype=torch.uint8)  # NaN where it is read before it is written
        assert call(ctypes.byref(a), ws.data_ptr(), n, stream) == 0
        torch.cuda.synchronize()
        assert (ws[n:] == 255).all()  # nothing behind what was asked for
    for x, y in zip(out, want):
        assert torch.equal(x, y)

    kp, vp = k[0, :200].contiguous(), v[0, :200].contiguous()
    for P, prefix in ((200, (kp, vp)), (3000, (kp.repeat(15, 1, 1), vp.repeat(15, 1, 1)))):
        want = fa.flash_attention_v100_shared_prefix(q[:, :3], *prefix, k, v, lens, softcap=11.0)
        out = torch.full((B, 3, H, D), float("nan"), device=DEV, dtype=torch.bfloat16)
        p = _ops.PrefixArgs()
        for n, t in zip(("q", "k_prefix", "v_prefix", "k", "v", "o"), (q, *prefix, k, v, out)):
            setattr(p, n, t.data_ptr())
            getattr(p, {"k_prefix": "kp", "v_prefix": "vp"}.get(n, n) + "_stride")[:] = t.stride()
        p.key_lengths = lens.data_ptr()
        (p.batch, p.seqlen_q, p.prefix_len, p.seqlen_k, p.num_heads, p.num_heads_kv, p.head_dim, p.dtype, p.scale,
         p.softcap) = B, 3, P, S, H, Hkv, D, 1, D ** -0.5, 11.0
        n = lib.fa_prefix_workspace_size(ctypes.byref(p))
        ws = torch.full((n + 256,), 255, device=DEV, dtype=torch.uint8)
        assert lib.fa_prefix_fwd(ctypes.byref(p), ws.data_ptr(), n, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (ws[n:] == 255).all()


@pytest.mark.parametrize("dt,D", [("bf16", 128), ("fp16", 80), ("fp32", 36), ("fp32", 128)])
@pytest.mark.parametrize("Sq,Sk", [(130, 130), (700, 70), (3, 500)])
def test_nothing_is_written_beside_the_outputs(dt, D, Sq, Sk):
    import ctypes

    lib, stream = _ops.load(), torch.cuda.current_stream().cuda_stream
    B, H, Hkv = 2, 4, 2
    q, k, v, do = make(B, Sq, Sk, H, Hkv, D, dt, seed=D)
    want = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = fa.flash_attention_v100_scored(*want, causal=True, query_offsets=Sk - Sq)
    want = [o.detach(), *torch.autograd.grad(o, want, do)]
    pad = 4 if dt == "fp32" else 8
    bufs = [torch.full((B + 1, t.shape[1] + 3, t.shape[2] + 1, D + pad), 7.0, device=DEV, dtype=t.dtype) for t in want]
    outs = [x[:B, :t.shape[1], :t.shape[2], :D] for x, t in zip(bufs, want)]
    lse = torch.full((B * H * Sq + 64,), 7.0, device=DEV)
    a = _ops.ScoredArgs()
    for n, t in zip(("q", "k", "v", "dout", "o", "dq", "dk", "dv"), (q, k, v, do, *outs)):
        setattr(a, n, t.data_ptr())
        getattr(a, ("do" if n == "dout" else n) + "_stride")[:] = t.stride()
    a.lse, a.query_offset, a.causal, a.scale = lse.data_ptr(), Sk - Sq, 1, D ** -0.5
    a.batch, a.seqlen_q, a.seqlen_k, a.num_heads, a.num_heads_kv, a.head_dim = B, Sq, Sk, H, Hkv, D
    a.dtype = {"fp16": 0, "bf16": 1, "fp32": 2}[dt]
    for size, call in ((lib.fa_scored_fwd_workspace_size, lib.fa_scored_fwd),
                       (lib.fa_scored_bwd_workspace_size, lib.fa_scored_bwd)):
        n = size(ctypes.byref(a))
        ws = torch.full((n + 256,), 255, device=DEV, dtype=torch.uint8)
        assert call(ctypes.byref(a), ws.data_ptr(), n, stream) == 0
        torch.cuda.synchronize()
        assert (ws[n:] == 255).all()
    for x, y, t in zip(bufs, outs, want):
        assert torch.equal(y, t)
        y.fill_(7.0)
        assert (x == 7.0).all()
    assert (lse[B * H * Sq:] == 7.0).all()
