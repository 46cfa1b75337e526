"""rotary_table_v100 and rotary_embedding_v100 against the 64-bit oracle."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make(B, S, H, D, dt, seed):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randn(B, S, H, D, generator=g).to(DT[dt]).to(DEV)


@pytest.mark.parametrize("kw", [{}, {"base": 500000.0}, {"scaling": "linear", "factor": 4.0},
                                {"scaling": "base", "factor": 8.0},
                                {"scaling": "ramp", "factor": 8.0, "original_positions": 4096}])
@pytest.mark.parametrize("R", [2, 20, 128])
def test_table(R, kw):
    n = 70000
    t = fa.rotary_table_v100(n, R, device=DEV, **kw)
    w, mul = oo.frequencies(R, kw.get("base", 10000.0), kw.get("scaling", "none"), kw.get("factor", 1.0),
                            kw.get("original_positions"))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * w
    ref = torch.cat([ang.cos(), ang.sin()], 1) * mul
    # one rounding to float32; w's own 64-bit rounding (some units) times the position
    tol = mul * (2.0 ** -24 + 2.0 ** -48 * torch.cat([ang, ang], 1))
    assert ((t.cpu().double() - ref).abs() <= tol).all()


def check(x, y, pos, w, mul, inter, inverse=False):
    ref, bound = oo.rotate(x, pos, w, mul, inter, inverse)
    oo.check({"y": y}, {"y": (ref, bound)}, ["y"], f"{tuple(x.shape)} {x.dtype} R={2 * w.numel()} {inter}")


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (64, 16), (80, 20), (80, 40), (96, 96), (33, 6), (256, 256),
                                 (130, 130), (2, 2), (31, 30)])
def test_layouts_types_and_gradients(D, R, inter, dt):
    B, S, H, Hkv = 2, 37, 5, 2
    table = fa.rotary_table_v100(64, R, device=DEV)
    w, mul = oo.frequencies(R)
    q, k = make(B, S, H, D, dt, 1).requires_grad_(True), make(B, S, Hkv, D, dt, 2).requires_grad_(True)
    gq, gk = make(B, S, H, D, dt, 3), make(B, S, Hkv, D, dt, 4)
    qo, ko = fa.rotary_embedding_v100(q, k, table, interleaved=inter)
    pos = torch.arange(S, device=DEV)
    check(q.detach(), qo.detach(), pos, w, mul, inter)
    check(k.detach(), ko.detach(), pos, w, mul, inter)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    check(gq, dq, pos, w, mul, inter, True)
    check(gk, dk, pos, w, mul, inter, True)


@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_positions(idt):
    B, S, R = 3, 50, 64
    table = fa.rotary_table_v100(1000, R, device=DEV)
    w, mul = oo.frequencies(R)
    g = torch.Generator("cpu").manual_seed(5)
    pos = torch.randint(0, 1000, (B, S), generator=g).to(idt).to(DEV)
    pos[1, 10:20] = -1
    pos[2, 3] = 999
    x = make(B, S, 4, 64, "bf16", 6)
    check(x, fa.rotary_embedding_v100(x, None, table, pos), pos, w, mul, False)
    check(x, fa.rotary_embedding_v100(x, None, table, pos.t().contiguous().t(), interleaved=True), pos, w, mul, True)
    check(x, fa.rotary_embedding_v100(x, None, table, pos[0]), pos[0], w, mul, False)
    # past the table: NaN in the rotated columns, never a read out of it
    far = pos.clone()
    far[0, 7], far[2, 1] = 1000, torch.iinfo(idt).max
    y = fa.rotary_embedding_v100(x, None, table[:, :], far)
    bad = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    bad[0, 7] = bad[2, 1] = True
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], fa.rotary_embedding_v100(x, None, table, pos)[~bad])


@pytest.mark.parametrize("inter", [False, True])
def test_in_place_and_strides(inter):
    B, S, H, Hkv, D, R = 2, 33, 6, 2, 96, 64
    table = fa.rotary_table_v100(S, R, device=DEV)
    qkv = make(B, S, H + 2 * Hkv, D, "fp16", 7)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hkv], qkv[:, :, H + Hkv:].clone()
    want = fa.rotary_embedding_v100(q, k, table, interleaved=inter)
    assert want[0].is_contiguous() and want[0].data_ptr() != q.data_ptr()
    got = fa.rotary_embedding_v100(q, k, table, interleaved=inter, inplace=True)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, :, H + Hkv:], v)  # the values beside them are left alone
    # transposed storage, odd offsets, no unit column stride, broadcast sequences
    w, mul = oo.frequencies(R)
    pos = torch.arange(S, device=DEV)
    for x in (make(B, H, S, D, "fp16", 8).transpose(1, 2), make(B, S, H, D + 3, "fp16", 9)[..., 3:],
              make(B, S, D, H, "fp16", 10).transpose(2, 3), make(1, S, H, D, "fp16", 11).expand(B, S, H, D)):
        check(x, fa.rotary_embedding_v100(x, None, table, interleaved=inter), pos, w, mul, inter)


def test_far_positions_and_scaling():
    # angles of some thousand turns and more: right to a rounding of the type
    n = 1 << 20
    table = fa.rotary_table_v100(n, 64, scaling="ramp", factor=16.0, original_positions=65536, device=DEV)
    w, mul = oo.frequencies(64, scaling="ramp", factor=16.0, original=65536)
    pos = torch.tensor([[n - 1, n - 2, 999983, 524287, 0]], device=DEV)
    x = make(1, 5, 3, 128, "fp32", 12)
    check(x, fa.rotary_embedding_v100(x, None, table, pos), pos, w, mul, False)


def test_sizes_from_one_token_to_many():
    for B, S, H, Hkv in ((1, 1, 1, 1), (16, 1, 32, 8), (1, 5000, 2, 1), (3, 700, 40, 40)):
        table = fa.rotary_table_v100(S, 64, device=DEV)
        w, mul = oo.frequencies(64)
        q, k = make(B, S, H, 64, "bf16", 13), make(B, S, Hkv, 64, "bf16", 14)
        qo, ko = fa.rotary_embedding_v100(q, k, table)
        pos = torch.arange(S, device=DEV)
        check(q, qo, pos, w, mul, False)
        check(k, ko, pos, w, mul, False)
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        x = torch.empty(shape, device=DEV, dtype=torch.bfloat16)
        assert fa.rotary_embedding_v100(x, None, table).shape == x.shape


def test_inner_products_depend_on_distance():
    # <R_m q, R_n k> is a function of m - n alone: the two sides' roundings are float32's
    table = fa.rotary_table_v100(4096, 64, device=DEV)
    q, k = make(1, 1, 1, 64, "fp32", 15), make(1, 1, 1, 64, "fp32", 16)

    def dot(m, n):
        a = fa.rotary_embedding_v100(q, None, table, torch.tensor([m], device=DEV))
        b = fa.rotary_embedding_v100(k, None, table, torch.tensor([n], device=DEV))
        return (a.double() * b.double()).sum().item()

    # each rotated value within 5 float32 roundings (bound of the oracle), twice over 64 products
    tol = 4 * 5 * 2.0 ** -24 * 2 * (q.abs().sum() * k.abs().sum()).item()
    for m, n in ((100, 37), (4000, 3937)):
        assert math.isclose(dot(m, n), dot(63, 0), abs_tol=tol)
