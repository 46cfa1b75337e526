"""Operators around attention, as a decoder's training step and its serving loop call them.

* ``scored``: attention whose scores are capped by a tanh, carry a bias that
  falls with the distance, or are masked by documents, prefixes and key lengths:
  training steps (forward, then the gradients of q, k, v and of learned slopes)
  and single new tokens over a cache;
* ``rotary``: rotary positions on q and k: training steps (forward and
  gradients), prefill of long scaled contexts, single tokens;
* ``shared``: new tokens of a batch of sequences that share a long prefix.

``run`` computes the plain form of each (elementary torch operations in 32
bits) or, with ``own``, calls the library.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _fa():
    root = os.path.join(os.getcwd(), "flash-attn-v100_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import flash_attention_v100
    return flash_attention_v100


# ---------------------------------------------------------------------------
# cases

def _scored(name, mode, B, Sq, Sk, H, Hkv, D, dtype, causal=True, cap=0.0, slopes=False, docs=0, prefix=0, lens=0,
            qk_std=1.0):
    """``docs``, ``prefix``, ``lens``: 0, or the number that the lengths of the
    documents, prefixes and filled caches are drawn from."""
    return {"name": name, "op": "scored", "mode": mode, "B": B, "Sq": Sq, "Sk": Sk, "H": H, "Hkv": Hkv, "D": D,
            "dtype": dtype, "causal": causal, "cap": cap, "slopes": slopes, "docs": docs, "prefix": prefix,
            "lens": lens, "qk_std": qk_std}


def _rotary(name, mode, B, S, H, Hkv, D, R, dtype, interleaved=False, scaling="none", factor=1.0, table=8192, docs=0):
    """``R``: rotated columns of the ``D``; ``table``: positions the program keeps."""
    return {"name": name, "op": "rotary", "mode": mode, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D, "R": R,
            "dtype": dtype, "interleaved": interleaved, "scaling": scaling, "factor": factor, "table": table,
            "docs": docs}


def _shared(name, B, Sq, P, Sk, H, Hkv, D, dtype, lens, cap=0.0, slopes=False):
    return {"name": name, "op": "shared", "mode": "token", "B": B, "Sq": Sq, "P": P, "Sk": Sk, "H": H, "Hkv": Hkv,
            "D": D, "dtype": dtype, "cap": cap, "slopes": slopes, "lens": lens}


def listed():
    return [
        # the smallest call: one new token of one sequence over a short cache, capped scores
        _scored("token_one", "token", 1, 1, 512, 8, 8, 64, "fp16", cap=30.0),
        # serving: one new token for each of 16 sequences over caches filled to different lengths, grouped heads
        _scored("token_cache", "token", 16, 1, 8192, 32, 8, 128, "bf16", cap=50.0, lens=11),
        # a training step with capped scores at 4096 tokens, grouped-query heads of 128
        _scored("cap_train", "train", 2, 4096, 4096, 32, 8, 128, "bf16", cap=30.0, qk_std=1.5),
        # a training step on sequences packed from documents, with a padded tail
        _scored("documents_train", "train", 2, 8192, 8192, 16, 16, 128, "bf16", docs=5),
        # a training step with a learned distance bias per head, a length that is no tile multiple
        _scored("distance_train", "train", 2, 1777, 1777, 12, 12, 64, "fp16", slopes=True),
        # full precision: a prefix read both ways, then causal text, head dim 80
        _scored("prefix_train_fp32", "train", 4, 700, 700, 12, 12, 80, "fp32", prefix=3),
        # decoding: q and k of one new token of 16 sequences, positions far into a context stretched 8 times
        _rotary("rotary_token", "token", 16, 1, 32, 8, 128, 128, "bf16", scaling="ramp", factor=8.0, table=65536),
        # a training step's positions on 4 x 4096 tokens, 32 heads of 128
        _rotary("rotary_train", "train", 4, 4096, 32, 32, 128, 128, "bf16"),
        # prefill of a long prompt of packed documents: neighbouring pairs, half of the head rotated
        _rotary("rotary_partial", "token", 1, 30001, 16, 4, 128, 64, "fp16", interleaved=True, scaling="linear",
                factor=4.0, table=32768, docs=7),
        # serving: 64 sequences after one 8192-token prompt, up to 512 keys of their own
        _shared("prefix_batch", 64, 1, 8192, 512, 32, 8, 128, "bf16", lens=13),
        # a small batch after a short prompt, capped scores and a distance bias
        _shared("prefix_small", 4, 1, 300, 40, 8, 8, 64, "fp16", lens=17, cap=30.0, slopes=True),
        # a few new tokens at once for each of 8 sequences after a long document, ragged sizes
        _shared("prefix_tokens", 8, 5, 20001, 1999, 16, 2, 128, "bf16", lens=19),
    ]


# what a drawn case may cost by its plain arithmetic (the largest listed case has 9.6e11) and hold in bytes
_MOST_FLOPS = {"fp16": 6e11, "bf16": 6e11, "fp32": 6e10}
_MOST_BYTES = 1.0e9


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    dt = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
    H = rng.choice([4, 8, 12, 16, 32])
    Hkv = rng.choice([H, H, H // 2, H // 4])
    seed = rng.randint(1, 10 ** 6)
    what = rng.choice(["train", "train", "token", "rotary", "shared"])
    if what == "train":
        S = _log(rng, 33, 8192)
        rule = rng.choice(["cap", "docs", "slopes", "prefix", "cap+slopes", "cap+docs", "docs+slopes"])
        return _scored("", "train", _log(rng, 1, 6), S, S, H, Hkv, rng.choice([32, 64, 64, 80, 96, 128, 128]), dt,
                       causal="prefix" in rule or rng.random() < 0.8, cap=rng.choice([20.0, 30.0, 50.0]) if "cap" in rule else 0.0,
                       slopes="slopes" in rule, docs=seed if "docs" in rule else 0,
                       prefix=seed if "prefix" in rule else 0, qk_std=rng.choice([1.0, 1.0, 1.5]))
    if what == "token":
        return _scored("", "token", _log(rng, 1, 48), rng.choice([1, 1, 1, rng.randint(2, 6)]), _log(rng, 100, 20000),
                       H, Hkv, rng.choice([64, 96, 128, 128]), dt, cap=rng.choice([0.0, 30.0, 50.0]),
                       slopes=rng.random() < 0.4, lens=seed)
    if what == "rotary":
        mode = rng.choice(["train", "token", "token"])
        D = rng.choice([32, 64, 80, 96, 128, 128])
        scaling = rng.choice(["none", "linear", "base", "ramp"])
        S = _log(rng, 1, 20000)
        return _rotary("", mode, _log(rng, 1, 32), S, H, Hkv, D, rng.choice([D, D, D // 2, D // 4]), dt,
                       interleaved=rng.random() < 0.5, scaling=scaling,
                       factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                       table=max(32768, S), docs=rng.choice([0, seed]))
    return _shared("", _log(rng, 2, 96), rng.choice([1, 1, 1, rng.randint(2, 6)]), _log(rng, 100, 24000),
                   _log(rng, 8, 2000), H, Hkv, rng.choice([64, 96, 128, 128]), dt, lens=seed,
                   cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3)


def draw(rng):
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["flops"] <= _MOST_FLOPS[c["dtype"]] and w["bytes"] <= _MOST_BYTES:
            del c["name"]
            return c


# ---------------------------------------------------------------------------
# lengths, from the case alone

def _documents(number, B, S):
    """Per sequence the lengths of its documents, log-uniform, and of a padded tail."""
    rng = random.Random(number)
    rows = []
    for _ in range(B):
        pad = rng.randint(0, S // 16)
        left, row = S - pad, []
        while left > 0:
            n = min(left, _log(rng, max(1, S // 64), max(2, S // 2)))
            row.append(n)
            left -= n
        rows.append((row, pad))
    return rows


def _prefixes(case):
    rng = random.Random(case["prefix"])
    return [rng.randint(0, case["Sk"] // 2) for _ in range(case["B"])]


def _lengths(case):
    """Filled keys of each sequence's cache, the new tokens among them."""
    if not case["lens"]:
        return [case["Sk"]] * case["B"]
    rng = random.Random(case["lens"])
    lo = min(case["Sk"], max(case["Sq"], case["Sk"] // 4))
    return [rng.randint(lo, case["Sk"]) for _ in range(case["B"])]


def _pairs(case):
    """(query, key) pairs that one head sees, over the batch."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    tri = lambda n: n * (n + 1) // 2  # noqa: E731
    if case["mode"] == "token":
        # query i of n keys sees n - Sq + i + 1 of them (none at a position before the first)
        return sum(sum(max(0, n - Sq + i + 1) for i in range(Sq)) for n in _lengths(case))
    if case["docs"]:
        return sum(tri(n) if case["causal"] else n * n for row, _ in _documents(case["docs"], B, Sk) for n in row)
    if not case["causal"]:
        return B * Sq * Sk
    if case["prefix"]:
        return sum(tri(Sk) + p * (p - 1) // 2 for p in _prefixes(case))
    return B * tri(Sk)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    if case["op"] == "rotary":
        # q and k read and written (twice in a training step), a table row a token
        cols = case["D"] * (H + Hkv)
        n = B * case["S"]
        rows = min(n, case["table"])
        passes = 2 if case["mode"] == "train" else 1
        return {"bytes": passes * (2 * n * cols * es + 4 * rows * case["R"]),
                "flops": passes * 3 * n * case["R"] * (H + Hkv)}
    Sq = case["Sq"]
    q_el = B * Sq * H * D
    if case["op"] == "shared":
        own_keys = sum(_lengths(case))
        pairs = _pairs(case) + B * Sq * case["P"]
        return {"bytes": es * (2 * q_el + 2 * (case["P"] + own_keys) * Hkv * D), "flops": 4 * D * H * pairs}
    pairs = _pairs(case)
    if case["mode"] == "token":
        return {"bytes": es * (2 * q_el + 2 * sum(_lengths(case)) * Hkv * D), "flops": 4 * D * H * pairs}
    kv_el = B * case["Sk"] * Hkv * D
    # q, o, do, dq and k, v, dk, dv
    return {"bytes": es * (4 * q_el + 4 * kv_el), "flops": 14 * D * H * pairs}


# ---------------------------------------------------------------------------
# inputs

def _frequencies(case, device):
    """Radians per position of each pair of columns, and the factor on cos and
    sin, in 64 bits."""
    R, base, f = case["R"], 10000.0, case["factor"]
    j = torch.arange(R // 2, device=device, dtype=torch.float64)
    if case["scaling"] == "base" and R > 2:
        base = base * f ** (R / (R - 2))
    inv = torch.exp(-(2.0 * j / R) * math.log(base))
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "ramp":
        # pairs that turn often over the original context keep their rate, slow ones are stretched
        turns = _original(case) * inv / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return inv * keep + inv / f * (1.0 - keep), 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _original(case):
    return max(1, int(case["table"] / case["factor"]))


def _doc_positions(case):
    return torch.cat([torch.arange(n, dtype=torch.int32) for row, pad in _documents(case["docs"], case["B"], case["S"])
                      for n in row + [pad]]).view(case["B"], case["S"])


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dt)

    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    st = {"case": case}
    if case["op"] == "rotary":
        S = case["S"]
        st["q"], st["k"] = randn(B, S, H, D), randn(B, S, Hkv, D)
        if case["mode"] == "train":
            st["dq"], st["dk"] = randn(B, S, H, D), randn(B, S, Hkv, D)
        if case["docs"]:
            pos = _doc_positions(case).cuda()
        elif S == 1:  # single tokens of sequences of any length
            pos = torch.randint(0, case["table"], (B, 1), generator=g, device="cuda", dtype=torch.int32)
        else:
            pos = torch.arange(S, device="cuda", dtype=torch.int32).repeat(B, 1)
        st["pos"] = pos
        return st
    Sq, Sk, std = case["Sq"], case["Sk"], case.get("qk_std", 1.0)
    st["q"], st["k"], st["v"] = randn(B, Sq, H, D, std=std), randn(B, Sk, Hkv, D, std=std), randn(B, Sk, Hkv, D)
    if case["mode"] == "train":
        st["do"] = randn(B, Sq, H, D)
    if case["op"] == "shared":
        st["kp"], st["vp"] = randn(case["P"], Hkv, D), randn(case["P"], Hkv, D)
    st["slopes"] = None
    if case["slopes"]:
        # geometric over the heads, as such biases are initialised, moved a little as after some training
        e = torch.arange(1, H + 1, device="cuda", dtype=torch.float32) * (-8.0 / H)
        st["slopes"] = torch.exp2(e) * (1.0 + 0.05 * torch.randn(H, generator=g, device="cuda"))
    st["docs"] = st["prefix"] = st["lens"] = None
    if case.get("docs"):
        st["docs"] = torch.stack([
            torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(row)]
                      + [torch.full((pad,), -1, dtype=torch.int32)])
            for row, pad in _documents(case["docs"], B, Sk)]).cuda()
    if case.get("prefix"):
        st["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
    if case["mode"] == "token":
        st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rotary":
        # the table of cosines and sines that a program builds once
        if own:
            kw = {}
            if case["scaling"] == "ramp":
                kw = {"original_positions": _original(case)}
            st["table"] = _fa().rotary_table_v100(case["table"], case["R"], scaling=case["scaling"],
                                                  factor=case["factor"], device="cuda", **kw)
        else:
            inv, mul = _frequencies(case, "cuda")
            ang = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * inv
            st["table"] = torch.cat([ang.cos() * mul, ang.sin() * mul], dim=1).float()
    elif own:
        _fa()
        if st["lens"] is not None and case["op"] == "scored":
            # position of the first new token: kept beside the lengths by a serving loop
            st["offsets"] = st["lens"] - case["Sq"]
        if case["mode"] == "train":
            for n in ("q", "k", "v") + (("slopes",) if case["slopes"] else ()):
                st[n].requires_grad_(True)
    if own and case["op"] == "rotary" and case["mode"] == "train":
        st["q"].requires_grad_(True)
        st["k"].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# the library's calls

def _run_own(st):
    fa, case = _fa(), st["case"]
    if case["op"] == "rotary":
        if case["mode"] == "train":
            q, k = fa.rotary_embedding_v100(st["q"], st["k"], st["table"], positions=st["pos"],
                                            interleaved=case["interleaved"])
            dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
            return q.detach(), k.detach(), dq, dk
        with torch.no_grad():
            return fa.rotary_embedding_v100(st["q"], st["k"], st["table"], positions=st["pos"],
                                            interleaved=case["interleaved"])
    if case["op"] == "shared":
        with torch.no_grad():
            return fa.flash_attention_v100_shared_prefix(st["q"], st["kp"], st["vp"], st["k"], st["v"],
                                                         key_lengths=st["lens"], softcap=case["cap"],
                                                         distance_slopes=st["slopes"])
    if case["mode"] == "token":
        with torch.no_grad():
            return fa.flash_attention_v100_scored(st["q"], st["k"], st["v"], causal=True, softcap=case["cap"],
                                                  distance_slopes=st["slopes"], key_lengths=st["lens"],
                                                  query_offsets=st["offsets"])
    o = fa.flash_attention_v100_scored(st["q"], st["k"], st["v"], causal=case["causal"], softcap=case["cap"],
                                       distance_slopes=st["slopes"], documents=st["docs"],
                                       prefix_lengths=st["prefix"])
    leaves = (st["q"], st["k"], st["v"]) + ((st["slopes"],) if case["slopes"] else ())
    return (o.detach(),) + torch.autograd.grad(o, leaves, st["do"])


# ---------------------------------------------------------------------------
# the plain form

def _plain_rotary(x, table, pos, R, interleaved, sign):
    t = table[pos.long()]  # (B, S, R)
    c, s = t[..., :R // 2].unsqueeze(2), t[..., R // 2:].unsqueeze(2) * sign
    xf = x.float()
    a, b = (xf[..., 0:R:2], xf[..., 1:R:2]) if interleaved else (xf[..., :R // 2], xf[..., R // 2:R])
    ya, yb = a * c - b * s, b * c + a * s
    rot = torch.stack([ya, yb], dim=-1).flatten(-2) if interleaved else torch.cat([ya, yb], dim=-1)
    return torch.cat([rot, xf[..., R:]], dim=-1).to(x.dtype)


def _scores(x, cap, dist, slope):
    """Capped and biased scores, and the cap's derivative."""
    der = None
    if cap:
        t = torch.tanh(x / cap)
        x, der = cap * t, 1.0 - t * t
    if slope is not None:
        x = x - slope * dist
    return x, der


def _soft(x, seen):
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(dim=-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    n = e.sum(dim=-1, keepdim=True)
    return e / torch.where(n == 0, torch.ones_like(n), n)


def _plain_train(st):
    """Forward and gradients, one (sequence, KV head) after the other."""
    case, q, k, v, do = st["case"], st["q"], st["k"], st["v"], st["do"]
    B, S, H, D = q.shape
    Hkv = k.shape[2]
    G, scale, cap = H // Hkv, D ** -0.5, case["cap"]
    o, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    dsl = torch.zeros(H, device=q.device) if case["slopes"] else None
    i = torch.arange(S, device=q.device)
    dist = (i[:, None] - i[None, :]).abs().float()
    for b in range(B):
        seen = torch.ones(S, S, dtype=torch.bool, device=q.device)
        if case["causal"]:
            seen = i[None, :] <= i[:, None]
            if st["prefix"] is not None:
                seen = seen | (i[None, :] < st["prefix"][b])
        if st["docs"] is not None:
            d = st["docs"][b]
            seen = seen & (d[:, None] == d[None, :]) & (d >= 0)[None, :]
        for n in range(Hkv):
            h = slice(n * G, (n + 1) * G)
            qh, doh = (t[b, :, h].transpose(0, 1).float() for t in (q, do))
            kh, vh = (t[b, :, n].float() for t in (k, v))
            slope = st["slopes"][h].view(G, 1, 1) if case["slopes"] else None
            x, der = _scores(torch.matmul(qh, kh.t()) * scale, cap, dist, slope)
            p = _soft(x, seen)
            oh = torch.matmul(p, vh)
            ds = p * (torch.matmul(doh, vh.t()) - (oh * doh).sum(-1, keepdim=True))
            if case["slopes"]:
                dsl[h] -= (ds * dist).sum(dim=(1, 2))
            dx = ds if der is None else ds * der
            o[b, :, h] = oh.transpose(0, 1).to(o.dtype)
            dq[b, :, h] = (torch.matmul(dx, kh) * scale).transpose(0, 1).to(q.dtype)
            dk[b, :, n] = (torch.matmul(dx.flatten(0, 1).t(), qh.flatten(0, 1)) * scale).to(k.dtype)
            dv[b, :, n] = torch.matmul(p.flatten(0, 1).t(), doh.flatten(0, 1)).to(v.dtype)
    return (o, dq, dk, dv) + ((dsl,) if case["slopes"] else ())


def _plain_token(st):
    """New tokens over each sequence's cache, and over a shared prefix before it."""
    case, q, k, v, lens = st["case"], st["q"], st["k"], st["v"], st["lens"].long()
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    G, scale = H // Hkv, D ** -0.5
    P = case["P"] if case["op"] == "shared" else 0
    # rows (i, g) of each sequence and KV head
    qh = q.float().view(B, Sq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Sq * G, D)
    kh, vh = (t.float().transpose(1, 2).contiguous() for t in (k, v))
    x = torch.matmul(qh, kh.transpose(-1, -2)) * scale
    if P:
        kp, vp = (st[n].float().transpose(0, 1).contiguous() for n in ("kp", "vp"))
        rows = qh.transpose(0, 1).reshape(Hkv, B * Sq * G, D)
        xp = torch.matmul(rows, kp.transpose(-1, -2)).view(Hkv, B, Sq * G, P).transpose(0, 1) * scale
        x = torch.cat([xp, x], dim=-1)
    pos = lens[:, None] - Sq + torch.arange(Sq, device=q.device)  # (B, Sq), own positions
    j = torch.arange(P + Sk, device=q.device) - P
    seen = (j <= pos[..., None]) & (pos[..., None] >= 0)
    seen = seen.repeat_interleave(G, dim=1)[:, None]  # (B, 1, Sq * G, P + Sk)
    dist = (pos[..., None] - j).abs().float().repeat_interleave(G, dim=1)[:, None]
    slope = None
    if st["slopes"] is not None:
        slope = st["slopes"].view(1, Hkv, 1, G, 1).expand(1, Hkv, Sq, G, 1).reshape(1, Hkv, Sq * G, 1)
    x, _ = _scores(x, case["cap"], dist, slope)
    p = _soft(x, seen)
    o = torch.matmul(p[..., P:].contiguous(), vh)
    if P:
        pp = p[..., :P].transpose(0, 1).reshape(Hkv, B * Sq * G, P)
        o = o + torch.matmul(pp, vp).view(Hkv, B, Sq * G, D).transpose(0, 1)
    return o.view(B, Hkv, Sq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Sq, H, D).to(q.dtype)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "rotary":
        R, il = case["R"], case["interleaved"]
        out = tuple(_plain_rotary(state[n], state["table"], state["pos"], R, il, 1.0) for n in ("q", "k"))
        if case["mode"] == "train":
            out += tuple(_plain_rotary(state[n], state["table"], state["pos"], R, il, -1.0) for n in ("dq", "dk"))
        return out
    return _plain_train(state) if case["mode"] == "train" else _plain_token(state)


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _exact_rotary(case, st):
    inv, mul = _frequencies(case, "cuda")
    turn = torch.polar(torch.full_like(inv, mul).expand(*st["pos"].shape, -1), st["pos"].double()[..., None] * inv)
    turn = turn.unsqueeze(2)  # (B, S, 1, R / 2)
    h = case["R"] // 2

    def rotate(x, w):
        y = x.double()
        first = torch.arange(h, device=x.device) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else h)
        z = torch.complex(y[..., first], y[..., second]) * w
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = (rotate(st["q"], turn), rotate(st["k"], turn))
    if case["mode"] == "train":
        out += (rotate(st["dq"], turn.conj()), rotate(st["dk"], turn.conj()))
    return out


def _exact_head(qh, kh, vh, qpos, kpos, hidden, cap, slope):
    """One head of one sequence: softmax over the keys that are not hidden."""
    s = qh @ kh.T / math.sqrt(qh.shape[1])
    if cap:
        e = torch.exp(-2.0 * (s / cap).abs())
        s = cap * torch.sign(s) * (1.0 - e) / (1.0 + e)
    if slope is not None:
        s = s - slope * (qpos[:, None] - kpos[None, :]).abs().double()
    empty = hidden.all(dim=1)
    s = torch.where(hidden, torch.full_like(s, -1e300), s)
    w = torch.softmax(s, dim=1)
    return torch.where(empty[:, None], torch.zeros_like(vh[:1]), w @ vh)


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, st)
    q, k, v = st["q"], st["k"], st["v"]
    B, Sq, H, D = q.shape
    G = H // k.shape[2]
    train = case["mode"] == "train"
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)] if train else []
    dsl = torch.zeros(H, dtype=torch.float64, device=q.device) if train and case["slopes"] else None
    P = case["P"] if case["op"] == "shared" else 0
    for b in range(B):
        n = int(st["lens"][b]) if st["lens"] is not None else case["Sk"]
        qpos = torch.arange(Sq, device=q.device) + (P + n - Sq if case["mode"] == "token" else 0)
        kpos = torch.arange(P + n, device=q.device)
        if train and not case["causal"]:
            hidden = torch.zeros(Sq, n, dtype=torch.bool, device=q.device)
        else:
            hidden = kpos[None, :] > qpos[:, None]
        if st["prefix"] is not None:
            hidden[:, :int(st["prefix"][b])] = False
        if st["docs"] is not None:
            d = st["docs"][b].tolist()
            dq, dk = (torch.tensor(x, device=q.device) for x in (d, [-2 if y < 0 else y for y in d]))
            hidden = hidden | (dq[:, None] != dk[None, :])
        if case["mode"] == "token":
            hidden[qpos < P] = True  # a token before the sequence's first
        for h in range(H):
            kh, vh = k[b, :n, h // G].double(), v[b, :n, h // G].double()
            if P:
                kh, vh = torch.cat([st["kp"][:, h // G].double(), kh]), torch.cat([st["vp"][:, h // G].double(), vh])
            leaves = [q[b, :, h].double(), kh, vh]
            slope = st["slopes"][h].double() if case["slopes"] else None
            if slope is not None:
                leaves.append(slope)
            if train:
                leaves = [t.detach().requires_grad_(True) for t in leaves]
            o = _exact_head(*leaves[:3], qpos, kpos, hidden, case["cap"], leaves[3] if slope is not None else None)
            out[b, :, h] = o.detach()
            if train:
                g = torch.autograd.grad(o, leaves, st["do"][b, :, h].double())
                grads[0][b, :, h] = g[0]
                grads[1][b, :, h // G] += g[1]
                grads[2][b, :, h // G] += g[2]
                if dsl is not None:
                    dsl[h] += g[3]
    if not train:
        return out
    return (out, *grads) + ((dsl,) if dsl is not None else ())
