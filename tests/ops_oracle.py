"""64-bit oracle of the operators around attention, with error bounds that follow
from the arithmetic of the kernels.

Per element every bound is a sum of products of magnitudes from the oracle
itself, each times the roundings on its path.  u = finfo(dtype).eps / 2 is one
rounding to the tensors' type, w = 2^-24 one of float32.

* a score: D products and sums (at most 2 w each: the matrix unit may cut
  instead of rounding) of magnitude scale sum |q||k|; the cap, as 1 - 2 r with
  r = 1 / (1 + 2^y), has a relative error of r of 2^-21 (exp2, addition and
  reciprocal at 1 to 2 ulps, with room for the argument's rounding) + 2^-22 |x| / cap, twice the
  cap's size; the bias and the conversions to log2 units a few w of their size.
* a probability: the score's error twice (its own and the largest of its row,
  through the sum), exp2 at 2^-22, its rounding to the type where it enters a product.
* a product over n terms: 2 n w of the sum of magnitudes; its rounding to the type.
* delta comes from the rounded output: its error is sum |dO| err(O).
"""
import math

import torch

W = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(val, err, dtype):
    """The bound `err` of a computed value near `val`, and its rounding to the type:
    half a step of what is rounded, |val| + err at most, or where that is below
    the normal numbers half of the smallest subnormal one (fp16: 2^-25)."""
    f = torch.finfo(dtype)
    return err + half_step(dtype) * (val.abs() + err) + f.tiny * f.eps / 2


def _heads(t, H):
    """(B, S, Hkv, D) -> (B, H, S, D) in 64 bits."""
    return t.double().transpose(1, 2).repeat_interleave(H // t.shape[2], dim=1)


def seen_mask(B, Sq, Sk, causal=False, documents=None, key_documents=None, prefix=None, lens=None, offsets=0,
              device="cpu"):
    """(B, Sq, Sk) booleans from the definition, one sequence after the other."""
    out = torch.zeros(B, Sq, Sk, dtype=torch.bool, device=device)
    i = torch.arange(Sq, device=device).view(Sq, 1)
    j = torch.arange(Sk, device=device).view(1, Sk)
    for b in range(B):
        off = int(offsets[b]) if isinstance(offsets, torch.Tensor) else int(offsets)
        s = (j < (int(lens[b]) if lens is not None else Sk)).expand(Sq, Sk)
        if causal:
            c = j <= i + off
            if prefix is not None:
                c = c | (j < int(prefix[b]))
            s = s & c
        if documents is not None:
            dq = documents.expand(B, Sq)[b].view(Sq, 1)
            dk = (documents if key_documents is None else key_documents).expand(B, Sk)[b].view(1, Sk)
            s = s & (dq == dk) & (dq >= 0)
        out[b] = s
    return out


def scored(q, k, v, do=None, scale=None, softcap=0.0, slopes=None, offsets=0, seen=None, kpos=None, qpos=None):
    """{name: (value, bound)} for o, lse and, with do, dq, dk, dv (and dslopes)."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    dev, dt = q.device, q.dtype
    u = half_step(dt)
    p_u = u if dt != torch.float32 else 0.0  # probabilities and dS enter products rounded to 16-bit types only
    p_0 = torch.finfo(dt).tiny * torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0  # where they are subnormal
    scale = D ** -0.5 if scale is None else scale
    qh, kh, vh = _heads(q, H), _heads(k, H), _heads(v, H)
    kt = kh.transpose(-1, -2).contiguous()
    x = qh @ kt * scale
    e_s = scale * (qh.abs() @ kt.abs()) * (2 * D * W)
    s, der, e_der = x, torch.ones_like(x), torch.zeros_like(x)
    if softcap:
        eps = 2.0 ** -21 + 2.0 ** -22 * (x.abs() / softcap)
        t = torch.tanh(x / softcap)
        r = (1 - t) / 2
        s, der = softcap * t, 1 - t * t
        e_s = e_s * der + e_s * e_s / softcap + softcap * (2 * r * eps + 2 * W)
        e_der = 4 * (1 - 2 * r).abs() * r * eps + 4 * W * der + 2 * e_s / softcap
    dist = None
    if slopes is not None:
        off = offsets.to(dev).view(B, 1) if isinstance(offsets, torch.Tensor) else offsets
        qp = (torch.arange(Sq, device=dev).view(1, Sq) + off).expand(B, Sq) if qpos is None else qpos
        kp = torch.arange(Sk, device=dev) if kpos is None else kpos
        dist = (qp.view(B, 1, Sq, 1) - kp.view(1, 1, 1, Sk)).abs().double()
        sl = slopes.double().view(-1, H, 1, 1)
        s = s - sl * dist
        e_s = e_s + sl.abs() * dist * (4 * W)
    e_s = e_s + s.abs() * (4 * W)
    hide = ~seen.to(dev).unsqueeze(1)
    s = s.masked_fill(hide, -math.inf)
    e_s = e_s.masked_fill(hide, 0.0)
    m = s.amax(-1, keepdim=True) if Sk else s.new_full((B, H, Sq, 1), -math.inf)
    empty = m == -math.inf
    m0 = torch.where(empty, torch.zeros_like(m), m)
    ex = torch.exp(s - m0)
    n = ex.sum(-1, keepdim=True)
    pr = ex / torch.where(empty, torch.ones_like(n), n)
    lse = torch.where(empty, m, m0 + n.log()).squeeze(-1)
    row = (e_s.amax(-1, keepdim=True) if Sk else torch.zeros_like(m)) + m0.abs() * (4 * W)
    e_p = e_s + row + 2.0 ** -21 + 2 * Sk * W  # relative error of a probability
    o = pr @ vh
    a = pr @ vh.abs()
    e_o = rounded(o, ((pr * (e_p + p_u) + p_0) @ vh.abs()) + a * (2 * Sk * W), dt)
    e_lse = row.squeeze(-1) + 2.0 ** -21 + 2 * Sk * W + torch.where(empty.squeeze(-1), torch.zeros_like(lse), lse).abs() * (4 * W)
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    res = {"o": (back(o), back(e_o)), "lse": (lse, e_lse)}
    if do is None:
        return res
    doh = _heads(do, H)
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
    e_dq = rounded(dq, scale * (e_dx @ kh.abs() + (dx.abs() @ kh.abs()) * (2 * Sk * W)), dt)
    dk = sum_kv(dxt @ qh) * scale
    e_dk = scale * (sum_kv(e_dx.transpose(-1, -2).contiguous() @ qh.abs()) + sum_kv(dxt.abs() @ qh.abs()) * rows)
    e_dk = rounded(dk, e_dk, dt)
    dv = sum_kv(ptr @ doh)
    e_dv = (sum_kv((pr * (e_p + p_u) + p_0).transpose(-1, -2).contiguous() @ doh.abs()) + sum_kv(ptr @ doh.abs()) * rows)
    e_dv = rounded(dv, e_dv, dt)
    res.update(dq=(back(dq), back(e_dq)), dk=(back(dk), back(e_dk)), dv=(back(dv), back(e_dv)))
    if slopes is not None:
        # the kernel sums P dP, |d| P and |d| P dP of a row in float32 and takes delta
        # from them: their errors, then a float32 per row
        e_pdp = (pr * (dp.abs() * (e_p + 2 * Sk * W + 2 * W) + e_dp))
        sdp, sd = (pr * dp).sum(-1), (pr * dist).sum(-1)
        e_row = ((e_pdp * dist).sum(-1) + e_pdp.sum(-1) * sd
                 + sdp.abs() * (pr * dist * (e_p + 2 * Sk * W + 2 * W)).sum(-1) + 4 * W * (sdp * sd).abs())
        g, e = -(ds * dist).sum((-1, -2)), e_row.sum(-1)
        if slopes.dim() == 1:
            g, e = g.sum(0), e.sum(0)
        res["dslopes"] = (g, e + 2 * W * g.abs())
    return res


def check(got, ref, names, label=""):
    """got: {name: tensor}; every element within its bound (equal infinities pass)."""
    lines, bad = [], []
    for n in names:
        val, bound = ref[n]
        x = got[n].double()
        assert x.shape == val.shape, (label, n, tuple(x.shape), tuple(val.shape))
        same = x == val
        err = torch.where(same, torch.zeros_like(val), (x - val).abs())
        ratio = torch.where(same, torch.zeros_like(val), err / (bound + 1e-30))
        worst = ratio.max().item() if ratio.numel() else 0.0
        lines.append(f"{label} {n}: error {err.max().item() if err.numel() else 0:.3e} at most {worst:.3f} of its bound")
        if not worst <= 1.0:  # a NaN fails too
            bad.append(lines[-1])
    print("\n".join(lines), flush=True)
    assert not bad, "\n".join(bad)


# ---------------------------------------------------------------------------
# rotary positions

def frequencies(R, base=10000.0, scaling="none", factor=1.0, original=None, low=1.0, high=32.0):
    """w_j in 64 bits, and the factor of cosines and sines of the ramp."""
    out = []
    for j in range(R // 2):
        b = base * factor ** (R / (R - 2)) if scaling == "base" and R > 2 else base
        w = b ** (-2.0 * j / R)
        if scaling == "linear":
            w /= factor
        if scaling == "ramp":
            g = min(1.0, max(0.0, (original * w / (2 * math.pi) - low) / (high - low)))
            w = w * g + w / factor * (1 - g)
        out.append(w)
    return torch.tensor(out, dtype=torch.float64), (0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0)


def rotate(x, pos, w, mul, interleaved, inverse=False):
    """Rotated x (B, S, H, D) in 64 bits and its bound: cosine and sine rounded
    to float32 (W each, and the angle's own error of 2^-52 of it), two products,
    a sum, one rounding to the type."""
    B, S, H, D = x.shape
    R = 2 * w.numel()
    y = x.double().clone()
    ang = pos.double().expand(B, S).view(B, S, 1, 1) * w.to(x.device)
    c, s = torch.cos(ang) * mul, torch.sin(ang) * mul * (-1 if inverse else 1)
    j = torch.arange(R // 2, device=x.device)
    ia, ib = (2 * j, 2 * j + 1) if interleaved else (j, j + R // 2)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    keep = (pos.expand(B, S) < 0).view(B, S, 1, 1)
    ya, yb = torch.where(keep, a, a * c - b * s), torch.where(keep, b, b * c + a * s)
    y[..., ia], y[..., ib] = ya, yb
    bound = torch.zeros_like(y)
    e = abs(mul) * (a.abs() + b.abs()) * (4 * W + 2.0 ** -50 * ang.abs())
    zero = torch.zeros_like(e)
    bound[..., ia] = torch.where(keep, zero, rounded(ya, e, x.dtype))
    bound[..., ib] = torch.where(keep, zero, rounded(yb, e, x.dtype))
    return y, bound
