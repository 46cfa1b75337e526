"""The operators around attention on a machine without a GPU: exports and struct
layouts of include/fa_ops.h, every status code of the checks (which make no
device call), workspace sizes, refusals of the Python entry points and the
layer's options."""
import copy
import ctypes
import os
import pickle
import re
import subprocess
import tempfile

import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100 import _lib, _ops
from flash_attention_v100.ops.rotary import _disjoint, _overlaps

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(REPO, "include")
HEADER = open(os.path.join(INC, "fa_ops.h")).read()
CODES = {n: int(v) for f in ("fa_abi.h", "fa_ops.h")
         for n, v in re.findall(r"#define (FA_(?:OK|ERR_\w+))\s+(-?\d+)", open(os.path.join(INC, f)).read())}
DT = {"fp16": 0, "bf16": 1, "fp32": 2}
STRUCTS = {"fa_scored_args": _ops.ScoredArgs, "fa_prefix_args": _ops.PrefixArgs, "fa_rotary_args": _ops.RotaryArgs}


def test_exports_are_the_headers():
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    declared = set(re.findall(r"^\s*(?:const\s+)?\w+\*?\s+\**(fa_\w+)\s*\(", text, flags=re.M))
    assert declared == set(_ops.EXPORTS)
    lib = _ops.load()
    assert lib.fa_ops_version() == _ops.OPS_VERSION
    assert all(hasattr(lib, n) for n in declared)


def test_struct_layouts():
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "fa_ops.h"', "int main(void) {"]
    for s, c in STRUCTS.items():
        lines.append(f'printf("{s} sizeof %zu\\n", sizeof({s}));')
        lines += [f'printf("{s} {f[0]} %zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_]
    lines += ['printf("dtypes f16 %d\\n", FA_DTYPE_F16); printf("dtypes bf16 %d\\n", FA_DTYPE_BF16);',
              'printf("dtypes f32 %d\\n", FA_DTYPE_F32);', "return 0; }"]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I", INC, "-o", exe, src], check=True)
        out = dict(ln.rsplit(" ", 1) for ln in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for s, c in STRUCTS.items():
        assert int(out[s + " sizeof"]) == ctypes.sizeof(c)
        for f in c._fields_:
            assert int(out[f"{s} {f[0]}"]) == getattr(c, f[0]).offset, (s, f[0])
    assert [int(out["dtypes " + n]) for n in ("f16", "bf16", "f32")] == [DT["fp16"], DT["bf16"], DT["fp32"]]


ADDR = 1 << 20  # looked at, never read


def strides(S, H, D):
    return (S * H * D, H * D, D, 1)


def scored_args(B=2, Sq=300, Sk=300, H=4, Hkv=2, D=64, dt="bf16"):
    a = _ops.ScoredArgs()
    for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, ADDR)
    for n in ("q", "o", "do", "dq"):
        getattr(a, n + "_stride")[:] = strides(Sq, H, D)
    for n in ("k", "v", "dk", "dv"):
        getattr(a, n + "_stride")[:] = strides(Sk, Hkv, D)
    a.batch, a.seqlen_q, a.seqlen_k, a.num_heads, a.num_heads_kv, a.head_dim, a.dtype = B, Sq, Sk, H, Hkv, D, DT[dt]
    a.scale = 0.125
    return a


def with_stride(name, i, v):
    def f(a):
        getattr(a, name)[i] = v
    return f


def with_(**kw):
    def f(a):
        for n, v in kw.items():
            setattr(a, n, v)
    return f


SCORED_BAD = [
    ("FA_ERR_SHAPE", with_(batch=-1)), ("FA_ERR_SHAPE", with_(seqlen_k=-1)), ("FA_ERR_DTYPE", with_(dtype=3)),
    ("FA_ERR_HEAD_DIM", with_(head_dim=0)), ("FA_ERR_HEAD_DIM", with_(head_dim=136)),
    ("FA_ERR_HEAD_DIM", with_(head_dim=60)), ("FA_ERR_HEADS", with_(num_heads=5)), ("FA_ERR_HEADS", with_(num_heads_kv=0)),
    ("FA_ERR_SCALE", with_(scale=0.0)), ("FA_ERR_SCALE", with_(scale=float("nan"))),
    ("FA_ERR_RULE", with_(softcap=-1.0)), ("FA_ERR_RULE", with_(softcap=float("inf"))),
    ("FA_ERR_RULE", with_(softcap=1e-7)), ("FA_ERR_RULE", with_(softcap=1e31)),
    ("FA_ERR_RULE", with_(slopes=ADDR, slopes_batch_stride=3)), ("FA_ERR_ALIGN", with_(slopes=ADDR + 2)),
    ("FA_ERR_RULE", with_(q_documents=ADDR)), ("FA_ERR_RULE", with_(k_documents=ADDR)),
    ("FA_ERR_RULE", with_(q_documents=ADDR, k_documents=ADDR, k_documents_stride=-1)),
    ("FA_ERR_ALIGN", with_(key_lengths=ADDR + 1)), ("FA_ERR_NULL_ARG", with_(q=None)),
    ("FA_ERR_NULL_ARG", with_(v=None)), ("FA_ERR_ALIGN", with_(k=ADDR + 8)), ("FA_ERR_ALIGN", with_(lse=ADDR + 2)),
    ("FA_ERR_STRIDE", with_stride("q_stride", 3, 2)), ("FA_ERR_STRIDE", with_stride("v_stride", 1, 65)),
    ("FA_ERR_STRIDE", with_stride("o_stride", 0, -64)), ("FA_ERR_TOO_LARGE", with_stride("k_stride", 0, 1 << 62)),
    ("FA_ERR_TOO_LARGE", with_(seqlen_q=2**31 - 1)),
]


@pytest.mark.parametrize("i", range(len(SCORED_BAD)))
def test_scored_refusals(i):
    code, change = SCORED_BAD[i]
    lib, a = _ops.load(), scored_args()
    assert lib.fa_scored_check(ctypes.byref(a), 0) == 0 and lib.fa_scored_check(ctypes.byref(a), 1) == 0
    change(a)
    for backward in (0, 1):
        assert lib.fa_scored_check(ctypes.byref(a), backward) == CODES[code]
    # the calls themselves refuse before any device work, and ask for no workspace
    assert lib.fa_scored_fwd(ctypes.byref(a), None, 0, None) == CODES[code]
    assert lib.fa_scored_bwd(ctypes.byref(a), None, 0, None) == CODES[code]
    assert lib.fa_scored_fwd_workspace_size(ctypes.byref(a)) == lib.fa_scored_bwd_workspace_size(ctypes.byref(a)) == 0


def test_scored_backward_refusals():
    lib = _ops.load()
    for code, change in (("FA_ERR_NULL_ARG", with_(dout=None)), ("FA_ERR_NULL_ARG", with_(lse=None)), ("FA_ERR_NULL_ARG", with_(dk=None)),
                         ("FA_ERR_STRIDE", with_stride("dv_stride", 2, 63)), ("FA_ERR_RULE", with_(dslopes=ADDR)),
                         ("FA_ERR_ALIGN", with_(slopes=ADDR, dslopes=ADDR + 2))):
        a = scored_args()
        change(a)
        assert lib.fa_scored_check(ctypes.byref(a), 0) == 0
        assert lib.fa_scored_check(ctypes.byref(a), 1) == CODES[code], code
    a = scored_args()
    need = lib.fa_scored_bwd_workspace_size(ctypes.byref(a))
    assert need > 0
    assert lib.fa_scored_bwd(ctypes.byref(a), None, need, None) == CODES["FA_ERR_WORKSPACE"]
    assert lib.fa_scored_bwd(ctypes.byref(a), ADDR, need - 1, None) == CODES["FA_ERR_WORKSPACE"]
    assert lib.fa_scored_bwd(ctypes.byref(a), ADDR + 16, need, None) == CODES["FA_ERR_WORKSPACE"]
    assert lib.fa_scored_check(None, 0) == CODES["FA_ERR_NULL_ARG"]


def test_workspace_sizes():
    lib = _ops.load()
    # forward: none without documents; with them the padded ids of every token and two ranges for 64 of them
    a = scored_args(B=1, Sq=1000, Sk=1000)
    assert lib.fa_scored_fwd_workspace_size(ctypes.byref(a)) == 0
    a.q_documents = a.k_documents = ADDR
    assert lib.fa_scored_fwd_workspace_size(ctypes.byref(a)) >= 1000 * 4
    # single tokens over a long cache: float32 parts of 128 columns, maximum and sum, for rows in units of 32
    a = scored_args(B=4, Sq=1, Sk=65536, H=8, Hkv=2, D=128)
    n = lib.fa_scored_fwd_workspace_size(ctypes.byref(a))
    assert n >= 2 * 4 * 2 * 32 * (128 + 2) * 4  # at least two parts of 4 x 2 units
    # small grids: float32 parts of dK and dV
    a = scored_args(B=1, Sq=2048, Sk=2048, H=8, Hkv=2, D=128)
    a.causal = 1
    assert lib.fa_scored_bwd_workspace_size(ctypes.byref(a)) >= 8 * 2 * 2 * 2048 * 128 * 4 + 2 * 8 * 2048 * 4


def prefix_args(B=3, Sq=2, P=500, Sk=40, H=4, Hkv=2, D=64, dt="bf16"):
    a = _ops.PrefixArgs()
    for n in ("q", "k_prefix", "v_prefix", "k", "v", "o", "lse"):
        setattr(a, n, ADDR)
    for n in ("q", "o"):
        getattr(a, n + "_stride")[:] = strides(Sq, H, D)
    for n in ("k", "v"):
        getattr(a, n + "_stride")[:] = strides(Sk, Hkv, D)
        getattr(a, n + "p_stride")[:] = (Hkv * D, D, 1)
    (a.batch, a.seqlen_q, a.prefix_len, a.seqlen_k, a.num_heads, a.num_heads_kv, a.head_dim, a.dtype,
     a.scale) = B, Sq, P, Sk, H, Hkv, D, DT[dt], 0.125
    return a


def test_prefix_refusals():
    lib = _ops.load()
    assert lib.fa_prefix_check(ctypes.byref(prefix_args())) == 0
    for code, change in (("FA_ERR_SHAPE", with_(prefix_len=-1)), ("FA_ERR_SHAPE", with_(seqlen_k=-1)),
                         ("FA_ERR_HEADS", with_(num_heads=3)), ("FA_ERR_DTYPE", with_(dtype=-1)),
                         ("FA_ERR_HEAD_DIM", with_(head_dim=160)), ("FA_ERR_SCALE", with_(scale=-1.0)),
                         ("FA_ERR_RULE", with_(softcap=float("nan"))), ("FA_ERR_NULL_ARG", with_(k_prefix=None)),
                         ("FA_ERR_NULL_ARG", with_(v=None)), ("FA_ERR_ALIGN", with_(v_prefix=ADDR + 4)),
                         ("FA_ERR_STRIDE", with_stride("kp_stride", 0, 100)), ("FA_ERR_STRIDE", with_stride("vp_stride", 2, 2)),
                         ("FA_ERR_ALIGN", with_(key_lengths=ADDR + 2))):
        a = prefix_args()
        change(a)
        assert lib.fa_prefix_check(ctypes.byref(a)) == CODES[code], code
        assert lib.fa_prefix_fwd(ctypes.byref(a), None, 0, None) == CODES[code], code
    a = prefix_args(P=5000)
    need = lib.fa_prefix_workspace_size(ctypes.byref(a))
    assert need > 0 and lib.fa_prefix_fwd(ctypes.byref(a), ADDR, need - 1, None) == CODES["FA_ERR_WORKSPACE"]
    a = prefix_args(B=0)
    assert lib.fa_prefix_fwd(ctypes.byref(a), None, 0, None) == 0  # no row: nothing to do


def rotary_args():
    a = _ops.RotaryArgs()
    for n in ("q", "q_out", "k", "k_out"):
        setattr(a, n, ADDR)
        getattr(a, n + "_stride")[:] = strides(10, 4, 64)
    a.table, a.table_positions = ADDR, 10
    a.batch, a.seqlen, a.num_heads, a.num_heads_k, a.head_dim, a.rotary_dim = 2, 10, 4, 4, 64, 64
    return a


def test_rotary_refusals():
    lib = _ops.load()
    assert lib.fa_rotary_check(ctypes.byref(rotary_args())) == 0
    for code, change in (("FA_ERR_SHAPE", with_(seqlen=-1)), ("FA_ERR_DTYPE", with_(dtype=9)),
                         ("FA_ERR_HEAD_DIM", with_(head_dim=0)), ("FA_ERR_HEAD_DIM", with_(head_dim=257)),
                         ("FA_ERR_ROTARY", with_(rotary_dim=3)), ("FA_ERR_ROTARY", with_(rotary_dim=66)),
                         ("FA_ERR_HEADS", with_(num_heads=0, num_heads_k=0)), ("FA_ERR_ROTARY", with_(table=None)),
                         ("FA_ERR_ROTARY", with_(table_positions=0)), ("FA_ERR_NULL_ARG", with_(k_out=None)),
                         ("FA_ERR_ALIGN", with_(q=ADDR + 1)), ("FA_ERR_STRIDE", with_stride("q_stride", 3, 2)),
                         ("FA_ERR_STRIDE", with_stride("k_out_stride", 1, 512)),  # in place, other rows
                         ("FA_ERR_ALIGN", with_(positions=ADDR + 4, positions_64=1)),
                         ("FA_ERR_TOO_LARGE", with_(batch=1 << 20, seqlen=1 << 20))):
        a = rotary_args()
        change(a)
        assert lib.fa_rotary_check(ctypes.byref(a)) == CODES[code], code
        assert lib.fa_rotary(ctypes.byref(a), None) == CODES[code], code
    for bad in ((0, 3, 0, 1e4, 1.0), (0, 64, 4, 1e4, 1.0), (0, 64, 0, -1.0, 1.0), (0, 64, 1, 1e4, float("inf"))):
        assert lib.fa_rotary_table(ADDR, 16, bad[1], bad[2], bad[3], bad[4], 1.0, 1.0, 32.0, 1.0, None) == CODES["FA_ERR_ROTARY"]


def test_messages_of_the_codes():
    lib = _lib.load()
    for n in ("FA_ERR_RULE", "FA_ERR_ROTARY"):
        assert b"unknown" not in lib.fa_strerror(CODES[n]).lower()


def test_host_module_refuses_other_versions():
    mod, lib = _ops.host(), _ops.load()
    addr = [ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.fa_ops_version, lib.fa_scored_fwd_workspace_size, lib.fa_scored_fwd, lib.fa_scored_bwd_workspace_size,
        lib.fa_scored_bwd, lib.fa_prefix_workspace_size, lib.fa_prefix_fwd, lib.fa_rotary)]
    sizes = [ctypes.sizeof(c) for c in (_ops.ScoredArgs, _ops.PrefixArgs, _ops.RotaryArgs)]
    other = ctypes.CFUNCTYPE(ctypes.c_int32)(lambda: _ops.OPS_VERSION + 1)
    with pytest.raises(RuntimeError):
        mod.bind_ops(ctypes.cast(other, ctypes.c_void_p).value, *sizes, *addr[1:])
    with pytest.raises(RuntimeError):
        mod.bind_ops(addr[0], sizes[0] + 8, *sizes[1:], *addr[1:])
    with pytest.raises((ValueError, RuntimeError)):
        mod.bind_ops(addr[0], *sizes, 0, *addr[2:])
    mod.bind_ops(addr[0], *sizes, *addr[1:])


# ---------------------------------------------------------------------------
# Python entry points: what they refuse without a GPU
def qkv(B=1, Sq=4, Sk=4, H=2, Hkv=2, D=8, dt=torch.float16):
    return torch.zeros(B, Sq, H, D, dtype=dt), torch.zeros(B, Sk, Hkv, D, dtype=dt), torch.zeros(B, Sk, Hkv, D, dtype=dt)


def test_no_cpu_path():
    q, k, v = qkv()
    for f in (lambda: fa.flash_attention_v100_scored(q, k, v), lambda: fa.rotary_embedding_v100(q, k, torch.zeros(4, 8)),
              lambda: fa.flash_attention_v100_shared_prefix(q, k[0], v[0], k, v), lambda: fa.rotary_table_v100(4, 8, device="cpu")):
        with pytest.raises(ValueError, match="no CPU path"):
            f()


@pytest.mark.parametrize("bad", [dict(q=torch.zeros(1, 4, 8)), dict(q=3), dict(v=torch.zeros(1, 5, 2, 8).half()),
                                 dict(q=torch.zeros(1, 4, 3, 8).half()), dict(q=torch.zeros(1, 4, 2, 8)),
                                 dict(q=torch.zeros(1, 4, 2, 8).int(), k=torch.zeros(1, 4, 2, 8).int(), v=torch.zeros(1, 4, 2, 8).int())])
def test_bad_qkv(bad):
    q, k, v = qkv()
    t = dict(dict(q=q, k=k, v=v), **bad)
    with pytest.raises((TypeError, ValueError)):
        fa.flash_attention_v100_scored(t["q"], t["k"], t["v"])
    with pytest.raises((TypeError, ValueError)):
        fa.flash_attention_v100_shared_prefix(t["q"], k[0], v[0], t["k"], t["v"])


@pytest.mark.parametrize("kw", [dict(scaling="other"), dict(max_positions=0), dict(max_positions=2.5), dict(rotary_dim=3),
                                dict(rotary_dim=0), dict(rotary_dim=258), dict(base=0.0), dict(base=float("inf")),
                                dict(factor=-1.0), dict(scaling="ramp"), dict(attention_factor=float("nan")),
                                dict(scaling="ramp", original_positions=64, low_rotations=4.0, high_rotations=4.0)])
def test_bad_tables(kw):
    kw = dict(dict(max_positions=8, rotary_dim=8, device="cpu"), **kw)
    with pytest.raises(ValueError) as e:
        fa.rotary_table_v100(kw.pop("max_positions"), kw.pop("rotary_dim"), **kw)
    assert "no CPU path" not in str(e.value)


def test_overlap_and_disjointness():
    x = torch.zeros(2, 5, 3, 4, 8)
    q, k, v = x.unbind(2)
    for t, over in ((q, False), (q[:, :, :1].expand(2, 5, 4, 8), True), (torch.zeros(8).expand(2, 5, 4, 8), True)):
        assert _overlaps(t.shape, t.stride()) == over
    assert _disjoint(q, k) and _disjoint(k, q) and _disjoint(q, v) and not _disjoint(q, q)
    y = torch.zeros(2, 5, 10, 8)
    assert _disjoint(y[:, :, :8], y[:, :, 8:]) and not _disjoint(y[:, :, :8], y[:, :, 7:9])
    assert _disjoint(y[:1], y[1:]) and not _disjoint(y, y[:, :, :2]) and not _disjoint(y[:, :, :2], y[:, 1:, :2][:, :4])
    assert _disjoint(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 1, 8))


# ---------------------------------------------------------------------------
# the layer's options
def test_layer_options_off_change_nothing():
    torch.manual_seed(0)
    a = fa.EnhancedMultiHeadAttention(64, 4)
    torch.manual_seed(0)
    b = fa.EnhancedMultiHeadAttention(64, 4, rotary_dim=16, softcap=30.0, distance_bias=True)
    assert list(a.state_dict()) == [n for n in b.state_dict() if n != "distance_slopes"]
    for n, p in a.named_parameters():
        assert torch.equal(p, b.state_dict()[n])
    assert torch.allclose(b.distance_slopes, torch.tensor([2.0 ** -2, 2.0 ** -4, 2.0 ** -6, 2.0 ** -8]))
    for bad in (3, 18, -2):
        with pytest.raises(ValueError, match="rotary_dim"):
            fa.EnhancedMultiHeadAttention(64, 4, rotary_dim=bad)


def test_layer_copies_and_older_pickles():
    m = fa.EnhancedMultiHeadAttention(64, 4, rotary_dim=16, distance_bias=True)
    m._tables["cuda:0"] = torch.zeros(1)
    c = copy.deepcopy(m)
    assert c._tables == {} and m._tables and torch.equal(c.distance_slopes, m.distance_slopes)
    p = pickle.loads(pickle.dumps(m))
    assert p._tables == {} and p.rotary_dim == 16
    old = dict(fa.EnhancedMultiHeadAttention(64, 4).__dict__)
    for n in ("rotary_dim", "rotary_base", "rotary_interleaved", "rotary_scaling", "max_positions", "softcap", "_tables"):
        del old[n]
    old["_parameters"] = {n: p for n, p in old["_parameters"].items() if n != "distance_slopes"}
    m = fa.EnhancedMultiHeadAttention.__new__(fa.EnhancedMultiHeadAttention)
    m.__setstate__(old)
    assert m.rotary_dim == 0 and m.softcap == 0.0 and m.distance_slopes is None


def test_layer_refusals():
    x = torch.zeros(2, 6, 64)
    for kw, call, match in ((dict(softcap=5.0, dropout=0.1), {}, "dropout"),
                            (dict(distance_bias=True), dict(attn_mask=torch.zeros(6, 6, dtype=torch.bool)), "attn_mask"),
                            (dict(softcap=5.0), dict(key_padding_mask=torch.zeros(2, 6)), "boolean"),
                            (dict(), dict(positions=torch.arange(6)), "rotary_dim"),
                            (dict(), dict(documents=torch.zeros(5, dtype=torch.int32)), "documents|no CPU path")):
        m = fa.EnhancedMultiHeadAttention(64, 4, **kw)
        with pytest.raises(ValueError, match=match):
            m(x, **call)
    m = fa.EnhancedMultiHeadAttention(64, 4)
    with pytest.raises(ValueError, match="one sequence"):
        m(x, x[:, :3], documents=torch.zeros(6, dtype=torch.int32))
