"""The paged cache on a machine without a GPU: exports and struct layouts of
include/fa_paged.h, every status code of the checks (which make no device call),
workspace sizes and the refusals of the Python entry points."""
import ctypes
import os
import re
import subprocess
import tempfile

import pytest
import torch

import flash_attention_v100 as fa
from flash_attention_v100 import _lib, _paged

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INC = os.path.join(REPO, "include")
HEADER = open(os.path.join(INC, "fa_paged.h")).read()
CODES = {n: int(v) for f in ("fa_abi.h", "fa_ops.h", "fa_paged.h")
         for n, v in re.findall(r"#define (FA_(?:OK|ERR_\w+))\s+(-?\d+)", open(os.path.join(INC, f)).read())}
STRUCTS = dict(zip(("fa_paged_args", "fa_cache_write_args", "fa_cache_accept_args", "fa_cache_fork_args",
                    "fa_cache_compact_args"), _paged.STRUCTS), fa_page_pool=_paged.PagePool)
ADDR = 1 << 20  # looked at, never read


def test_exports_are_the_headers():
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    declared = set(re.findall(r"^\s*(?:const\s+)?\w+\*?\s+\**(fa_\w+)\s*\(", text, flags=re.M))
    assert declared == set(_paged.EXPORTS)
    lib = _paged.load()
    assert lib.fa_paged_version() == _paged.PAGED_VERSION
    for name, value in (("FA_MAX_TREE_NODES", _paged.MAX_TREE_NODES), ("FA_PAGED_VERSION", _paged.PAGED_VERSION)):
        assert re.search(rf"#define {name} {value}\b", HEADER)
    assert "FA_MAX_POOL_PAGES (1 << 20)" in HEADER and _paged.MAX_POOL_PAGES == 1 << 20
    assert _lib.strerror(CODES["FA_ERR_PAGES"]) != _lib.strerror(-99)
    assert len(set(CODES.values())) == len(CODES)


def test_struct_layouts():
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "fa_paged.h"', "int main(void) {"]
    for s, c in STRUCTS.items():
        lines.append(f'printf("{s} sizeof %zu\\n", sizeof({s}));')
        lines += [f'printf("{s} {f[0]} %zu\\n", offsetof({s}, {f[0]}));' for f in c._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "l.c"), os.path.join(d, "l")
        open(src, "w").write("\n".join(lines + ["return 0; }"]))
        subprocess.run(["gcc", "-I", INC, "-o", exe, src], check=True)
        out = dict(ln.rsplit(" ", 1) for ln in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for s, c in STRUCTS.items():
        assert int(out[s + " sizeof"]) == ctypes.sizeof(c)
        for f in c._fields_:
            assert int(out[f"{s} {f[0]}"]) == getattr(c, f[0]).offset, (s, f[0])


def pool(batch=3, pages=40, size=16, Hkv=2, D=64, dtype=1, layers=1, cols=5, table=True, lens=True):
    c = _paged.PagePool()
    st = (pages * size * Hkv * D, size * Hkv * D, Hkv * D, D, 1)
    c.k, c.v = ADDR, 2 * ADDR
    c.k_stride, c.v_stride = (ctypes.c_int64 * 5)(*st), (ctypes.c_int64 * 5)(*st)
    c.layers, c.pages, c.page_size, c.num_heads_kv, c.head_dim, c.dtype, c.batch = layers, pages, size, Hkv, D, dtype, batch
    c.table_cols, c.page_table, c.table_stride = (cols, 3 * ADDR, cols) if table else (1, None, 0)
    c.key_lengths = 4 * ADDR if lens else None
    return c


def paged_args(N=4, H=4, **kw):
    a = _paged.PagedArgs()
    a.pool = pool(**kw)
    D = a.pool.head_dim
    st = (ctypes.c_int64 * 4)(N * H * D, H * D, D, 1)
    a.q, a.o, a.q_stride, a.o_stride = 5 * ADDR, 6 * ADDR, st, st
    a.seqlen_q, a.num_heads, a.scale, a.softcap = N, H, 0.125, 0.0
    return a


def write_args(N=4, **kw):
    a = _paged.CacheWriteArgs()
    a.pool = pool(**kw)
    c = a.pool
    st = (ctypes.c_int64 * 5)(c.batch * N * c.num_heads_kv * c.head_dim, N * c.num_heads_kv * c.head_dim,
                              c.num_heads_kv * c.head_dim, c.head_dim, 1)
    a.k, a.v, a.k_stride, a.v_stride, a.tokens = 5 * ADDR, 6 * ADDR, st, st, N
    return a


def accept_args(**kw):
    a = _paged.CacheAcceptArgs()
    a.pool = pool(**kw)
    a.path, a.path_stride, a.path_cols, a.tokens, a.new_lengths = 5 * ADDR, 6, 6, 9, 6 * ADDR
    return a


def fork_args(new_batch=7, **kw):
    a = _paged.CacheForkArgs()
    a.pool = pool(**kw)
    a.sources, a.more, a.more_all, a.new_batch, a.new_table, a.new_lengths = 5 * ADDR, None, 1, new_batch, 6 * ADDR, 7 * ADDR
    return a


def compact_args(**kw):
    a = _paged.CacheCompactArgs()
    a.pool = pool(**kw)
    a.new_table, a.used = 5 * ADDR, 6 * ADDR
    return a


CHECKS = {"fa_paged": paged_args, "fa_cache_write": write_args, "fa_cache_accept": accept_args,
          "fa_cache_fork": fork_args, "fa_cache_compact": compact_args}


def status(name, a):
    return getattr(_paged.load(), name + "_check")(ctypes.byref(a))


def put(a, path, value):
    *head, last = path.split(".")
    for h in head:
        a = getattr(a, h)
    if "[" in last:
        last, i = last[:-1].split("[")
        getattr(a, last)[int(i)] = value
    else:
        setattr(a, last, value)


@pytest.mark.parametrize("name", CHECKS)
@pytest.mark.parametrize("path,value,code", [
    ("pool.layers", 0, "FA_ERR_SHAPE"), ("pool.pages", -1, "FA_ERR_SHAPE"), ("pool.page_size", -16, "FA_ERR_SHAPE"),
    ("pool.batch", -1, "FA_ERR_SHAPE"), ("pool.table_cols", -1, "FA_ERR_SHAPE"), ("pool.dtype", 3, "FA_ERR_DTYPE"),
    ("pool.head_dim", 0, "FA_ERR_HEAD_DIM"), ("pool.head_dim", 129, "FA_ERR_HEAD_DIM"), ("pool.head_dim", 60, "FA_ERR_HEAD_DIM"),
    ("pool.num_heads_kv", 0, "FA_ERR_HEADS"), ("pool.num_heads_kv", 1 << 17, "FA_ERR_TOO_LARGE"),
    ("pool.layers", 1 << 15, "FA_ERR_TOO_LARGE"), ("pool.page_size", 24, "FA_ERR_PAGES"), ("pool.page_size", 8, "FA_ERR_PAGES"),
    ("pool.page_size", 0, "FA_ERR_PAGES"), ("pool.page_table", 3 * ADDR + 2, "FA_ERR_ALIGN"),
    ("pool.table_stride", -1, "FA_ERR_PAGES"), ("pool.table_cols", 1 << 24, "FA_ERR_TOO_LARGE"),
    ("pool.key_lengths", 4 * ADDR + 1, "FA_ERR_ALIGN"), ("pool.k", None, "FA_ERR_NULL_ARG"), ("pool.v", 2 * ADDR + 8, "FA_ERR_ALIGN"),
    ("pool.k_stride[4]", 2, "FA_ERR_STRIDE"), ("pool.v_stride[2]", 3, "FA_ERR_STRIDE"), ("pool.k_stride[1]", -64, "FA_ERR_STRIDE"),
    ("pool.v_stride[0]", 1 << 41, "FA_ERR_TOO_LARGE"), ("pool.k_stride[2]", 1 << 23, "FA_ERR_TOO_LARGE")])
def test_pool_codes(name, path, value, code):
    a = CHECKS[name]()
    assert status(name, a) == CODES["FA_OK"]
    put(a, path, value)
    assert status(name, a) == CODES[code]


@pytest.mark.parametrize("name,path,value,code", [
    ("fa_paged", "q", None, "FA_ERR_NULL_ARG"), ("fa_paged", "o", 6 * ADDR + 4, "FA_ERR_ALIGN"),
    ("fa_paged", "q_stride[1]", 7, "FA_ERR_STRIDE"), ("fa_paged", "num_heads", 5, "FA_ERR_HEADS"),
    ("fa_paged", "num_heads", 0, "FA_ERR_HEADS"), ("fa_paged", "seqlen_q", -1, "FA_ERR_SHAPE"),
    ("fa_paged", "scale", 0.0, "FA_ERR_SCALE"), ("fa_paged", "softcap", -1.0, "FA_ERR_RULE"),
    ("fa_paged", "softcap", 1e-9, "FA_ERR_RULE"), ("fa_paged", "slopes", ADDR + 1, "FA_ERR_ALIGN"),
    ("fa_paged", "lse", ADDR + 2, "FA_ERR_ALIGN"), ("fa_paged", "parents", ADDR + 2, "FA_ERR_ALIGN"),
    ("fa_paged", "pool.layers", 2, "FA_ERR_SHAPE"),
    ("fa_cache_write", "k", None, "FA_ERR_NULL_ARG"), ("fa_cache_write", "v_stride[3]", 7, "FA_ERR_STRIDE"),
    ("fa_cache_write", "tokens", -1, "FA_ERR_SHAPE"), ("fa_cache_write", "tokens", 1 << 30, "FA_ERR_TOO_LARGE"),
    ("fa_cache_accept", "path", None, "FA_ERR_NULL_ARG"), ("fa_cache_accept", "new_lengths", None, "FA_ERR_NULL_ARG"),
    ("fa_cache_accept", "new_lengths", 4 * ADDR, "FA_ERR_PAGES"), ("fa_cache_accept", "path_stride", -1, "FA_ERR_PAGES"),
    ("fa_cache_accept", "path_cols", -1, "FA_ERR_SHAPE"), ("fa_cache_accept", "path", 5 * ADDR + 1, "FA_ERR_ALIGN"),
    ("fa_cache_fork", "sources", None, "FA_ERR_NULL_ARG"), ("fa_cache_fork", "new_table", None, "FA_ERR_NULL_ARG"),
    ("fa_cache_fork", "new_table", 3 * ADDR, "FA_ERR_PAGES"), ("fa_cache_fork", "new_lengths", 4 * ADDR, "FA_ERR_PAGES"),
    ("fa_cache_fork", "new_batch", -1, "FA_ERR_SHAPE"), ("fa_cache_fork", "new_batch", 1 << 30, "FA_ERR_TOO_LARGE"),
    ("fa_cache_fork", "more", 9, "FA_ERR_ALIGN"), ("fa_cache_fork", "pool.page_table", None, "FA_ERR_NULL_ARG"),
    ("fa_cache_fork", "pool.pages", (1 << 20) + 1, "FA_ERR_PAGES"),
    ("fa_cache_compact", "used", None, "FA_ERR_NULL_ARG"), ("fa_cache_compact", "new_table", 3 * ADDR, "FA_ERR_PAGES"),
    ("fa_cache_compact", "pool.page_table", None, "FA_ERR_NULL_ARG"), ("fa_cache_compact", "used", 3, "FA_ERR_ALIGN"),
    ("fa_cache_compact", "pool.pages", (1 << 20) + 1, "FA_ERR_PAGES")])
def test_own_codes(name, path, value, code):
    a = CHECKS[name]()
    put(a, path, value)
    assert status(name, a) == CODES[code]


def test_trees_and_rows_of_tokens():
    a = paged_args(N=257)
    assert status("fa_paged", a) == 0
    a.parents = ADDR
    assert status("fa_paged", a) == CODES["FA_ERR_PAGES"]
    a = paged_args(table=False)
    assert status("fa_paged", a) == 0
    a.pool.page_size = 33
    assert status("fa_paged", a) == 0
    a.pool.pages = 2
    assert status("fa_paged", a) == CODES["FA_ERR_PAGES"]
    a.pool.pages, a.pool.table_cols = 3, 2
    assert status("fa_paged", a) == CODES["FA_ERR_PAGES"]


def test_grids_that_no_launch_takes():
    # 2^32 threads a grid: units of 32 rows of 256, rows of 64 of 4 rows, forks of 256 each
    a = paged_args(N=2000, H=4, Hkv=4, cols=1, batch=65535)    # 63 units of each of 4 heads: 16.5 million, below 2^24
    assert status("fa_paged", a) == 0
    a = paged_args(N=2100, H=4, Hkv=4, cols=1, batch=65535)    # 66: 17.3 million
    assert status("fa_paged", a) == CODES["FA_ERR_TOO_LARGE"]
    a = write_args(N=1 << 10)
    a.pool.batch = 1 << 17
    assert status("fa_cache_write", a) == 0
    a.pool.batch = 1 << 18
    assert status("fa_cache_write", a) == CODES["FA_ERR_TOO_LARGE"]
    a = fork_args(new_batch=(1 << 24) - 1)
    assert status("fa_cache_fork", a) == 0
    a.new_batch += 1
    assert status("fa_cache_fork", a) == CODES["FA_ERR_TOO_LARGE"]
    # pieces of 16 KB of all layers of a page, in 31 bits
    a = compact_args()
    a.pool.page_size, a.pool.num_heads_kv, a.pool.layers = 1 << 14, 1 << 9, 1 << 11
    assert status("fa_cache_compact", a) == 0
    a.pool.layers = 1 << 12
    assert status("fa_cache_compact", a) == CODES["FA_ERR_TOO_LARGE"]


def test_workspaces_and_refusals_before_any_launch():
    lib = _paged.load()
    size = lib.fa_paged_workspace_size
    assert size(ctypes.byref(paged_args(cols=32))) == 0            # up to 512 tokens: units are not shared
    big = paged_args(cols=64)
    n = size(ctypes.byref(big))
    assert n > 0 and n % 256 == 0
    assert lib.fa_paged_fwd(ctypes.byref(big), None, 0, None) == CODES["FA_ERR_WORKSPACE"]
    assert lib.fa_paged_fwd(ctypes.byref(big), ADDR, n - 1, None) == CODES["FA_ERR_WORKSPACE"]
    assert lib.fa_paged_fwd(ctypes.byref(big), ADDR + 4, n, None) == CODES["FA_ERR_WORKSPACE"]
    for name, make in (("fa_cache_fork", fork_args), ("fa_cache_compact", compact_args)):
        a = make()
        n = getattr(lib, name + "_workspace_size")(ctypes.byref(a))
        assert n > 0
        for ws, b in ((None, n), (ADDR, n - 1), (ADDR + 8, n)):
            assert getattr(lib, name)(ctypes.byref(a), ws, b, None) == CODES["FA_ERR_WORKSPACE"]
    # nothing to do: no launch (there is no device here)
    for name, make in CHECKS.items():
        if name == "fa_cache_compact":
            continue
        a = make(new_batch=0) if name == "fa_cache_fork" else make(batch=0)
        run = getattr(lib, "fa_paged_fwd" if name == "fa_paged" else name)
        assert (run(ctypes.byref(a), None, 0, None) if name in ("fa_paged", "fa_cache_fork") else run(ctypes.byref(a), None)) == 0
    assert lib.fa_cache_write(ctypes.byref(write_args(N=0)), None) == 0
    assert lib.fa_paged_fwd(ctypes.byref(paged_args(N=0)), None, 0, None) == 0


def test_bind_refuses_other_layouts():
    lib, mod = _paged.load(), _paged.host()
    addr = [ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.fa_paged_version, lib.fa_paged_workspace_size, lib.fa_paged_fwd, lib.fa_cache_write, lib.fa_cache_accept,
        lib.fa_cache_fork_workspace_size, lib.fa_cache_fork, lib.fa_cache_compact_workspace_size, lib.fa_cache_compact)]
    sizes = [ctypes.sizeof(s) for s in _paged.STRUCTS]
    mod.bind_paged(addr[0], *sizes, *addr[1:])
    for i in range(5):
        with pytest.raises(RuntimeError, match="version"):
            mod.bind_paged(addr[0], *[s + 8 * (j == i) for j, s in enumerate(sizes)], *addr[1:])
    other = ctypes.CFUNCTYPE(ctypes.c_int32)(lambda: _paged.PAGED_VERSION + 1)
    with pytest.raises(RuntimeError, match="version"):
        mod.bind_paged(ctypes.cast(other, ctypes.c_void_p).value, *sizes, *addr[1:])
    with pytest.raises(ValueError, match="null"):
        mod.bind_paged(addr[0], *sizes, *addr[1:-1], 0)
    with pytest.raises(TypeError):
        mod.bind_paged(addr[0])


def test_entry_points_need_a_gpu_and_tensors():
    kc, vc, q = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64), torch.zeros(1, 1, 2, 64)
    t, n, k = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 2, 64)
    calls = [lambda: fa.flash_attention_v100_paged(q, kc, vc, n, t), lambda: fa.paged_cache_write_v100(k, k, kc, vc, n, t),
             lambda: fa.paged_cache_accept_v100(kc, vc, n, t, 1, t), lambda: fa.paged_cache_fork_v100(kc, vc, t, n, n),
             lambda: fa.paged_cache_compact_v100(kc, vc, t, n)]
    for c in calls:
        with pytest.raises(ValueError, match="GPU"):
            c()
    for c in (lambda: fa.flash_attention_v100_paged(None, kc, vc, n, t), lambda: fa.flash_attention_v100_paged(q, None, vc, n, t),
              lambda: fa.paged_cache_write_v100(None, k, kc, vc, n, t), lambda: fa.paged_cache_accept_v100(kc, vc, n, None, 1, t),
              lambda: fa.paged_cache_fork_v100(kc, vc, None, n, n), lambda: fa.paged_cache_compact_v100(kc, vc, None, n)):
        with pytest.raises(TypeError):
            c()
    with pytest.raises(ValueError, match="4-dim"):
        fa.flash_attention_v100_paged(q[0], kc, vc, n, t)
    with pytest.raises(ValueError, match="2-dim"):
        fa.paged_cache_accept_v100(kc, vc, n, n, 1, t)


def test_oracle_trees():
    import paged_oracle as po

    assert po.ancestors([-1, 0, 0, 1, -2, 4, 9, 7]) == [[0], [0, 1], [0, 2], [0, 1, 3], [], [], [], []]
    kc = torch.arange(2 * 48.0).view(1, 6, 16, 1, 1)
    out = po.fork(kc, kc, [[0, 1], [2, -1]], [20, 3], [0, 0, 1], [1, 13, 1])
    assert out[2:] == ([[0, 1], [-1, -1], [2, -1]], [21, 0, 4])
