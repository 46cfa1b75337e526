"""Calls of the operators around attention at the edge of what they document, as far
as a machine without a GPU shows it."""
import ctypes
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as ad

import flash_attention_v100 as fa
from flash_attention_v100 import _ops, modules
from flash_attention_v100.ops import scored
from test_ops_cpu import ADDR, CODES, prefix_args, scored_args


def test_forward_mode_derivatives_are_refused():
    # before anything else is looked at: without the refusal the result has no tangent
    q, k, v = (torch.zeros(1, 4, 2, 8) for _ in range(3))
    table = torch.zeros(4, 8)
    for f, args in ((fa.flash_attention_v100_scored, (q, k, v)), (fa.rotary_embedding_v100, (q, k, table)),
                    (lambda q, k, v: fa.flash_attention_v100_shared_prefix(q, k[0], v[0], k, v), (q, k, v))):
        for i in range(len(args)):
            with ad.dual_level(), torch.no_grad():
                dual = [ad.make_dual(t, torch.ones_like(t)) if n == i else t for n, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*dual)
                with ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="no CPU path"):
                    f(*dual)
            with pytest.raises(ValueError, match="no CPU path"):
                f(*args)


def fake_tables(monkeypatch):
    """rotary_table_v100 of the layer on the CPU: its arguments, in order of the calls."""
    calls = []

    def table(n, dim, base, device=None, **kw):
        calls.append((n, dim, base, tuple(sorted(kw.items()))))
        return torch.zeros(n, dim)

    monkeypatch.setattr(modules, "rotary_table_v100", table)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(synchronize=lambda: None))
    return calls


def test_layer_table_of_inference_mode_serves_training(monkeypatch):
    calls = fake_tables(monkeypatch)
    m = fa.EnhancedMultiHeadAttention(64, 4, rotary_dim=16)
    with torch.inference_mode():
        t = m._rotary_table(torch.device("cpu"))
    assert not t.is_inference()
    assert m._rotary_table(torch.device("cpu")) is t and len(calls) == 1


def test_layer_table_follows_the_options(monkeypatch):
    calls = fake_tables(monkeypatch)
    cpu = torch.device("cpu")
    m = fa.EnhancedMultiHeadAttention(64, 4, rotary_dim=16, max_positions=32)
    t = m._rotary_table(cpu)
    for change in (lambda: setattr(m, "max_positions", 64), lambda: setattr(m, "rotary_base", 500.0),
                   lambda: setattr(m, "rotary_dim", 8), lambda: m.rotary_scaling.update(scaling="linear", factor=2.0)):
        change()
        u = m._rotary_table(cpu)
        assert u is not t and m._rotary_table(cpu) is u
        t = u
    assert calls == [(32, 16, 1e4, ()), (64, 16, 1e4, ()), (64, 16, 500.0, ()), (64, 8, 500.0, ()),
                     (64, 8, 500.0, (("factor", 2.0), ("scaling", "linear")))]
    # an earlier table is kept: a captured graph may read it
    assert len(m._tables) == 5
    m.rotary_dim, m.rotary_base, m.max_positions, m.rotary_scaling = 16, 1e4, 32, {}
    m._rotary_table(cpu)
    assert len(calls) == 5


@pytest.mark.parametrize("Sq,Sk,q_ids,k_ids", [(0, 5, None, ADDR), (5, 0, ADDR, None), (0, 0, None, None),
                                               (0, 5, ADDR, None), (5, 5, None, None)])
def test_documents_of_empty_sides(Sq, Sk, q_ids, k_ids):
    # an empty tensor's address is null: no sign of a missing array
    lib, a = _ops.load(), scored_args(Sq=Sq, Sk=Sk)
    a.q_documents, a.k_documents = q_ids, k_ids
    for backward in (0, 1):
        assert lib.fa_scored_check(ctypes.byref(a), backward) == 0
    assert lib.fa_scored_fwd_workspace_size(ctypes.byref(a)) == 0
    a.seqlen_q = a.seqlen_k = 5
    assert lib.fa_scored_check(ctypes.byref(a), 0) == (CODES["FA_ERR_RULE"] if (q_ids is None) != (k_ids is None) else 0)


def test_lse_near_is_checked():
    lib, a = _ops.load(), scored_args()
    for lse_near, code in ((ADDR, 0), (ADDR + 2, CODES["FA_ERR_ALIGN"])):
        a.lse_near = lse_near
        for backward in (0, 1):
            assert lib.fa_scored_check(ctypes.byref(a), backward) == code


def test_scale_past_the_cap_is_refused():
    # scale / softcap past float32 would make a score of 0 a NaN
    lib = _ops.load()
    for scale, cap, ok in ((1e30, 1e-6, True), (3e38, 1e-6, False), (3e38, 100.0, True), (3e38, 0.0, True)):
        a = scored_args()
        a.scale, a.softcap = scale, cap
        assert lib.fa_scored_check(ctypes.byref(a), 0) == (0 if ok else CODES["FA_ERR_RULE"])
        p = prefix_args()
        p.scale, p.softcap = scale, cap
        assert lib.fa_prefix_check(ctypes.byref(p)) == (0 if ok else CODES["FA_ERR_RULE"])
    assert scored.check_softcap(1e-6, 1e30) == 1e-6
    with pytest.raises(ValueError, match="scale"):
        scored.check_softcap(1e-6, 3e38)
