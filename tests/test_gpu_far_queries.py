"""Queries far from their keys: the distance to the nearest of them is common to a
row and leaves no trace in its outputs and gradients, within bounds that grow with
the spread of the distances only."""
import ctypes

import pytest
import torch

import flash_attention_v100 as fa
import ops_edges_oracle as eo
import ops_oracle as oo
from flash_attention_v100 import _ops
from ops_edges_oracle import DEV, make, train

pytestmark = pytest.mark.gpu


FAR = [8192, 65536, 1 << 20, (1 << 24) + 3, (1 << 28) + 1, 1 << 30]


def forward(q, k, v, slopes, off, label, lens=None, **kw):
    got = dict(zip(("o", "lse"), fa.flash_attention_v100_scored(
        q, k, v, query_offsets=off, distance_slopes=slopes, key_lengths=lens, return_softmax_lse=True, **kw)))
    seen = oo.seen_mask(q.shape[0], q.shape[1], k.shape[1], kw.get("causal", False), None, None, None, lens, off, DEV)
    oo.check(got, eo.scored(q, k, v, None, 0.0, slopes, off, seen, lens), ["o", "lse"], label)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("off", FAR)
def test_far_queries(off, D, dt):
    q, k, v, _ = make(2, 170, 500, 4, 2, D, dt, seed=off % 1000)
    slopes = torch.tensor([0.5, 0.0625, 0.01, 0.001], device=DEV)
    forward(q, k, v, slopes, off, f"{off} D={D} {dt}", causal=True)
    forward(q, k, v, slopes, -off, f"{-off} D={D} {dt}")


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_offsets_inside_and_outside(dt):
    q, k, v, _ = make(4, 130, 300, 2, 1, 64, dt, seed=7)
    off = torch.tensor([1 << 20, 200, -5, 100000], dtype=torch.int32, device=DEV)
    lens = torch.tensor([300, 120, 300, 1], dtype=torch.int32, device=DEV)
    slopes = torch.tensor([[0.1, -0.004], [0.02, 0.3], [0.5, 0.0], [0.001, 1.0]], device=DEV)
    forward(q, k, v, slopes, off, dt, lens)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("off", FAR)
def test_few_far_queries(off, dt):
    # the few-row kernel: one part a row, and parts that are joined
    slopes = torch.tensor([0.5, 0.0625, 0.01, 0.001], device=DEV)
    for Sq, Sk in ((2, 100), (5, 5000)):
        q, k, v, _ = make(2, Sq, Sk, 4, 2, 64, dt, seed=Sq)
        forward(q, k, v, slopes, off, f"{Sq} x {Sk}, {off} {dt}", causal=True)
        forward(q, k, v, slopes, -off, f"{Sq} x {Sk}, {-off} {dt}")


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("off", FAR)
def test_slopes_of_far_queries(off, D, dt):
    q, k, v, do = make(2, 70, 500, 4, 2, D, dt, seed=off % 1000)
    slopes = torch.tensor([0.5, 0.0625, 0.01, 0.001], device=DEV)
    train(q, k, v, do, f"offset {off} D={D} {dt}", causal=True, query_offsets=off, distance_slopes=slopes)
    train(q, k, v, do, f"offset {-off} D={D} {dt}", query_offsets=-off, distance_slopes=slopes)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_slopes_of_far_queries_of_other_calls(dt):
    # offsets and lengths of each sequence (one inside the keys, one before the
    # first), a cap, slopes of each sequence, negative ones too
    q, k, v, do = make(4, 130, 300, 2, 1, 64, dt, seed=7)
    off = torch.tensor([1 << 20, 200, -5, 100000], dtype=torch.int32, device=DEV)
    lens = torch.tensor([300, 120, 300, 1], dtype=torch.int32, device=DEV)
    slopes = torch.tensor([[0.1, -0.004], [0.02, 0.3], [0.5, 0.0], [0.001, 1.0]], device=DEV)
    for kw in ({}, {"softcap": 20.0}):
        train(q, k, v, do, f"{kw} {dt}", query_offsets=off, key_lengths=lens, distance_slopes=slopes, **kw)
    # a grid of one group of waves a block
    q, k, v, do = make(5, 500, 300, 30, 30, 64, dt, seed=8)
    slopes = torch.exp2(-8.0 * torch.arange(1, 31, device=DEV) / 30)
    train(q, k, v, do, f"one group {dt}", causal=True, query_offsets=1 << 20, distance_slopes=slopes)


def c_calls(q, k, v, do, slopes, off, out, causal=0, forward=True):
    """fa_scored_fwd (unless o and the LSEs are given) and fa_scored_bwd; out: name -> tensor."""
    lib, stream = _ops.load(), torch.cuda.current_stream().cuda_stream
    a = _ops.ScoredArgs()
    for n, t in dict(q=q, k=k, v=v, dout=do, **{n: out[n] for n in ("o", "dq", "dk", "dv")}).items():
        setattr(a, n, t.data_ptr())
        getattr(a, ("do" if n == "dout" else n) + "_stride")[:] = t.stride()
    for n in ("lse", "lse_near", "dslopes"):
        setattr(a, n, out[n].data_ptr() if n in out else None)
    a.slopes, a.query_offset, a.causal = slopes.data_ptr(), off, causal
    (a.batch, a.seqlen_q, a.seqlen_k, a.num_heads, a.num_heads_kv, a.head_dim, a.dtype,
     a.scale) = q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], 2, q.shape[3] ** -0.5
    calls = [(lib.fa_scored_fwd_workspace_size, lib.fa_scored_fwd)] if forward else []
    for size, call in calls + [(lib.fa_scored_bwd_workspace_size, lib.fa_scored_bwd)]:
        n = size(ctypes.byref(a))
        ws = torch.empty(n + 256, device=DEV, dtype=torch.uint8)
        assert call(ctypes.byref(a), ws.data_ptr(), n, stream) == 0


@pytest.mark.parametrize("off", [100000, 1 << 24, 1 << 30])
def test_c_entries_with_the_lse_of_the_nearest_key(off):
    B, Sq, Sk, H, D = 1, 40, 300, 2, 64
    q, k, v, do = make(B, Sq, Sk, H, H, D, "fp32", seed=3)
    slopes = torch.tensor([0.5, 0.25], device=DEV)
    out = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("dslopes", slopes))}
    out["lse"], out["lse_near"] = torch.zeros(2, B, H, Sq, device=DEV)
    c_calls(q, k, v, do, slopes, off, out)
    ref = eo.scored(q, k, v, do, 0.0, slopes, off, oo.seen_mask(B, Sq, Sk, device=DEV))
    oo.check(out, ref, ["o", "lse", "dq", "dk", "dv", "dslopes"], str(off))


@pytest.mark.parametrize("causal", [0, 1])
def test_gradients_of_a_part_of_the_keys(causal):
    # o and the LSE of a whole row, the keys in two parts: P is e^(s - LSE) as given,
    # dq adds up, dk and dv are the parts'
    B, S, H, D, n = 2, 300, 2, 64, 130
    q, k, v, do = make(B, S, S, H, H, D, "fp32", seed=4)
    slopes = torch.tensor([0.05, 0.002], device=DEV)
    new = lambda: {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}  # noqa: E731
    whole = new()
    whole["lse"] = torch.zeros(B, H, S, device=DEV)
    c_calls(q, k, v, do, slopes, 0, whole, causal)
    parts = []
    for a, b in ((0, n), (n, S)):
        out = new()
        out.update(o=whole["o"], lse=whole["lse"], dk=torch.zeros_like(k[:, a:b]), dv=torch.zeros_like(v[:, a:b]))
        c_calls(q, k[:, a:b], v[:, a:b], do, slopes, -a, out, causal, forward=False)
        parts.append(out)
    got = dict(whole, dq=parts[0]["dq"] + parts[1]["dq"], **{n: torch.cat([p[n] for p in parts], 1) for n in ("dk", "dv")})
    ref = oo.scored(q, k, v, do, None, 0.0, slopes, 0, oo.seen_mask(B, S, S, bool(causal), device=DEV))
    oo.check(whole, ref, ["o", "lse", "dq", "dk", "dv"], "whole")
    # one more rounding where the two parts of dq meet
    ref["dq"] = (ref["dq"][0], ref["dq"][1] + 2 * oo.W * ref["dq"][0].abs())
    oo.check(got, ref, ["dq", "dk", "dv"], "parts")
