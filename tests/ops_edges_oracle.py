"""64-bit oracle of scored attention at its edges: caps far above the scores, and
queries far from their keys.  As tests/ops_oracle.py, but with bounds that grow
neither with the cap nor with the distance of a query to the keys.

u is one rounding to the tensors' type, W = 2^-24 one of float32.

* cap: cap tanh(x / cap) is computed with a relative error of 2^-20 at most: the
  constants scale / cap and cap log2 e, two products (W each, 4 W), and tanh by a
  series (2e-8 of it) below 0.45, by 1 - 2 r above, where it is at least 0.42 and
  r's error 2^-21 r with r below 0.29: 2 * 0.29 * 2^-21 / 0.42 < 1.4 * 2^-21.
  Its derivative 1 - t^2 has twice the error of t^2 and one rounding.
* distances: the softmax of a row does not change when all of its distances lose
  the one to the nearest key that exists, p = clamp(i + off, 0, len - 1), so
  the scores' errors are those of slope |p - j|, and only the LSE holds
  slope |i + off - p|.
* the slopes' gradient of a row, sum_j |p - j| dS: the errors of dS where delta
  may be off by any error common to the row (sum_j dS is made 0 again), times |p - j|.
"""
import math

import torch

import flash_attention_v100 as fa
import ops_oracle as oo

W = oo.W
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def scored(q, k, v, do=None, softcap=0.0, slopes=None, offsets=0, seen=None, lens=None):
    """{name: (value, bound)}, as ops_oracle.scored."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    dev, dt = q.device, q.dtype
    u = oo.half_step(dt)
    p_u = u if dt != torch.float32 else 0.0
    p_0 = torch.finfo(dt).tiny * torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0
    scale = D ** -0.5
    qh, kh, vh = oo._heads(q, H), oo._heads(k, H), oo._heads(v, H)
    kt = kh.transpose(-1, -2).contiguous()
    x = qh @ kt * scale
    e_s = scale * (qh.abs() @ kt.abs()) * (2 * D * W)
    s, der, e_der = x, torch.ones_like(x), torch.zeros_like(x)
    if softcap:
        t = torch.tanh(x / softcap)
        s, der = softcap * t, 1 - t * t
        e_der = 2 * t * t * 2.0 ** -20 + 2 * W + 2 * t.abs() * e_s / softcap
        e_s = e_s + s.abs() * 2.0 ** -20
    ref = torch.zeros(B, H, Sq, 1, device=dev, dtype=torch.float64)
    dist = None
    if slopes is not None:
        off = offsets.to(dev).view(B, 1) if isinstance(offsets, torch.Tensor) else offsets
        qp = (torch.arange(Sq, device=dev).view(1, Sq) + off).expand(B, Sq)
        last = (torch.full((B,), Sk, device=dev) if lens is None else lens.to(dev)).view(B, 1) - 1
        p = torch.minimum(qp.clamp_min(0), last.clamp_min(0))
        sl = slopes.double().view(-1, H, 1, 1)
        dist = (p.view(B, 1, Sq, 1) - torch.arange(Sk, device=dev)).abs().double()
        ref = sl * (qp - p).abs().double().view(B, 1, Sq, 1)
        s = s - sl * dist
        e_s = e_s + sl.abs() * dist * (4 * W)
    e_s = e_s + s.abs() * (4 * W)
    hide = ~seen.to(dev).unsqueeze(1)
    s, e_s = s.masked_fill(hide, -math.inf), e_s.masked_fill(hide, 0.0)
    m = s.amax(-1, keepdim=True)
    empty = m == -math.inf
    m0 = torch.where(empty, torch.zeros_like(m), m)
    ex = torch.exp(s - m0)
    n = ex.sum(-1, keepdim=True)
    pr = ex / torch.where(empty, torch.ones_like(n), n)
    sums = (2 * seen.to(dev).sum(-1).double() + 4).view(B, 1, Sq, 1) * W  # of the keys seen: the others add zeros
    row = e_s.amax(-1, keepdim=True) + m0.abs() * (4 * W)
    e_p = e_s + row + 2.0 ** -21 + 2 * sums
    lse = torch.where(empty, m, m0 + n.log() - ref).squeeze(-1)
    e_lse = (row + 2.0 ** -21 + sums + ref.abs() * (4 * W)).squeeze(-1) + torch.where(
        empty.squeeze(-1), torch.zeros_like(lse), lse).abs() * (4 * W)
    o = pr @ vh
    e_o = oo.rounded(o, ((pr * (e_p + p_u) + p_0) @ vh.abs()) + (pr @ vh.abs()) * sums, dt)
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    res = {"o": (back(o), back(e_o)), "lse": (lse, e_lse)}
    if do is None:
        return res
    doh = oo._heads(do, H)
    vt = vh.transpose(-1, -2).contiguous()
    dp = doh @ vt
    e_dp = (doh.abs() @ vt.abs()) * (2 * D * W)
    delta = (pr * dp).sum(-1, keepdim=True)
    e_delta = (doh.abs() * e_o).sum(-1, keepdim=True) + (doh.abs() * o.abs()).sum(-1, keepdim=True) * (2 * D * W)
    ds = pr * (dp - delta)
    e_ds = ds.abs() * (e_p + 4 * W) + pr * (e_dp + e_delta + (dp.abs() + delta.abs()) * W)
    dx = ds * der
    e_dx = e_ds * der + ds.abs() * e_der + dx.abs() * p_u + p_0
    ptr, dxt = pr.transpose(-1, -2).contiguous(), dx.transpose(-1, -2).contiguous()
    sum_kv = lambda t: t.view(B, Hkv, H // Hkv, Sk, D).sum(2)  # noqa: E731
    rows = 2 * Sq * (H // Hkv) * W
    dq = dx @ kh * scale
    e_dq = oo.rounded(dq, scale * (e_dx @ kh.abs() + (dx.abs() @ kh.abs()) * sums), dt)
    dk = sum_kv(dxt @ qh) * scale
    e_dk = scale * (sum_kv(e_dx.transpose(-1, -2).contiguous() @ qh.abs()) + sum_kv(dxt.abs() @ qh.abs()) * rows)
    dv = sum_kv(ptr @ doh)
    e_dv = sum_kv((pr * (e_p + p_u) + p_0).transpose(-1, -2).contiguous() @ doh.abs()) + sum_kv(ptr @ doh.abs()) * rows
    res.update(dq=(back(dq), back(e_dq)), dk=(back(dk), back(oo.rounded(dk, e_dk, dt))),
               dv=(back(dv), back(oo.rounded(dv, e_dv, dt))))
    if slopes is not None:
        # P (dP - delta') with a delta' off by e_delta at most, which the row's sum takes out again
        pds = pr * ((dp - delta).abs() + e_delta)
        e_pds = pds * (e_p + 4 * W + sums) + pr * (e_dp + (dp.abs() + delta.abs()) * W)
        sd = (pr * dist).sum(-1)
        e_row = ((e_pds * dist).sum(-1) + e_pds.sum(-1) * sd
                 + e_delta.squeeze(-1) * (pr * dist * (e_p + 4 * W + sums)).sum(-1)
                 + 8 * W * (pds * dist).sum(-1) + 8 * W * e_delta.squeeze(-1) * sd)
        g, e = -(ds * dist).sum((-1, -2)), e_row.sum(-1)
        if slopes.dim() == 1:
            g, e = g.sum(0), e.sum(0)
        res["dslopes"] = (g, e + 2 * W * g.abs())
    return res


def make(B, Sq, Sk, H, Hkv, D, dt, seed=0):
    g = torch.Generator("cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DT[dt]).to(DEV)  # noqa: E731
    return r(B, Sq, H, D), r(B, Sk, Hkv, D), r(B, Sk, Hkv, D), r(B, Sq, H, D)


def train(q, k, v, do, label, **kw):
    """One step's outputs and gradients within the bounds of the edges' oracle."""
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    names = ["o", "lse", "dq", "dk", "dv"]
    leaves = [q, k, v]
    slopes = kw.get("distance_slopes")
    if slopes is not None:
        kw["distance_slopes"] = slopes = slopes.detach().requires_grad_(True)
        leaves.append(slopes)
        names.append("dslopes")
    o, lse = fa.flash_attention_v100_scored(q, k, v, return_softmax_lse=True, **kw)
    got = dict(zip(names, (o.detach(), lse) + torch.autograd.grad(o, leaves, do)))
    off = kw.get("query_offsets")
    off = 0 if off is None else off
    seen = oo.seen_mask(q.shape[0], q.shape[1], k.shape[1], kw.get("causal", False), kw.get("documents"),
                        kw.get("key_documents"), kw.get("prefix_lengths"), kw.get("key_lengths"), off, DEV)
    ref = scored(q.detach(), k.detach(), v.detach(), do, kw.get("softcap") or 0.0,
                 None if slopes is None else slopes.detach(), off, seen, kw.get("key_lengths"))
    oo.check(got, ref, names, label)
