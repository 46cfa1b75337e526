"""Calls of the operators around attention at the edge of what they document: tokens
that keep their bits, forward-mode derivatives, empty sides, layers that were used
without gradients first."""
import math

import pytest
import torch

import flash_attention_v100 as fa
from ops_edges_oracle import DEV, DT, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 16), (33, 6), (31, 30)])
def test_tokens_at_negative_positions_keep_their_bits(D, R, inter, dt):
    B, S, H = 2, 20, 3
    x = torch.randn(B, S, H, D, generator=torch.Generator("cpu").manual_seed(5)).to(DT[dt]).to(DEV)
    pos = torch.arange(S, device=DEV).repeat(B, 1)
    pos[0, 3:9] = -1
    pos[1] = -7
    out = pos < 0
    vals = torch.tensor([math.inf, -0.0, 1.0, math.nan, -math.inf, 0.0, -2.0], device=DEV).to(DT[dt])
    pad = vals[torch.arange(H * D, device=DEV) % 7].view(H, D)
    x[out] = pad
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    table = fa.rotary_table_v100(64, R, device=DEV)
    before = x.view(bits).clone()
    x.requires_grad_(True)
    y = fa.rotary_embedding_v100(x, None, table, pos, interleaved=inter)
    assert torch.equal(y.detach().view(bits)[out], before[out])
    g, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(g.view(bits)[out], before[out])
    x = x.detach().clone()
    z = fa.rotary_embedding_v100(x, None, table, pos, interleaved=inter, inplace=True)
    assert z is x or z.data_ptr() == x.data_ptr()
    assert torch.equal(x.view(bits), y.detach().view(bits))


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as ad

    q, k, v, _ = make(1, 4, 4, 2, 2, 64, "fp32")
    slopes = torch.ones(2, device=DEV)
    table = fa.rotary_table_v100(8, 64, device=DEV)
    calls = {
        "scored": (lambda q, k, v, s: fa.flash_attention_v100_scored(q, k, v, distance_slopes=s), (q, k, v, slopes)),
        "shared": (lambda q, kp, vp, k, v, s: fa.flash_attention_v100_shared_prefix(q, kp, vp, k, v, distance_slopes=s),
                   (q, k[0], v[0], k, v, slopes)),
        "rotary": (lambda q, k: fa.rotary_embedding_v100(q, k, table)[0], (q, k)),
        "rotary, one": (lambda q: fa.rotary_embedding_v100(q, None, table, inplace=True), (q,)),
    }
    for name, (f, args) in calls.items():
        for i in range(len(args)):
            with ad.dual_level(), torch.no_grad():
                dual = [ad.make_dual(t, torch.ones_like(t)) if n == i else t for n, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*dual)
                ad.unpack_dual(f(*args))  # a level without duals changes nothing
        print(name, "refused", flush=True)


def test_layer_trains_after_inference_mode():
    torch.manual_seed(3)
    m = fa.EnhancedMultiHeadAttention(64, 2, rotary_dim=16, softcap=20.0).to(DEV).half()
    x = torch.randn(2, 30, 64, device=DEV, dtype=torch.half)
    with torch.inference_mode():
        a = m(x, is_causal=True)[0]
    y = m(x, is_causal=True)[0]
    assert torch.equal(a, y)
    y.sum().backward()
    assert m.q_proj.weight.grad is not None


def test_layer_follows_its_rotary_options():
    torch.manual_seed(4)
    kw = dict(rotary_dim=16, rotary_base=500.0, rotary_scaling={"scaling": "linear", "factor": 2.0}, max_positions=64)
    m = fa.EnhancedMultiHeadAttention(64, 2, rotary_dim=16, max_positions=32).to(DEV).half()
    n = fa.EnhancedMultiHeadAttention(64, 2, **kw).to(DEV).half()
    n.load_state_dict(m.state_dict())
    x = torch.randn(1, 50, 64, device=DEV, dtype=torch.half)
    with torch.no_grad():
        m(x[:, :30])
        m.rotary_base, m.max_positions = 500.0, 64
        m.rotary_scaling.update(kw["rotary_scaling"])
        assert torch.equal(m(x, is_causal=True)[0], n(x, is_causal=True)[0])


@pytest.mark.parametrize("Sq,Sk", [(0, 5), (5, 0), (0, 0), (0, 300), (300, 0)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_documents_of_empty_sides(Sq, Sk, dt):
    q, k, v, do = make(2, Sq, Sk, 2, 1, 64, dt)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    s = torch.ones(2, device=DEV).requires_grad_(True)
    for idt in (torch.int32, torch.int64):
        ids = lambda n: torch.zeros(2, n, dtype=idt, device=DEV)  # noqa: E731
        o, lse = fa.flash_attention_v100_scored(q, k, v, documents=ids(Sq), key_documents=ids(Sk), distance_slopes=s,
                                                return_softmax_lse=True)
        assert o.shape == q.shape and not o.any() and (lse == -math.inf).all()
        for g in torch.autograd.grad(o, (q, k, v, s), do):
            assert not g.any()
