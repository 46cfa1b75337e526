"""The paged cache's entry points at their edges: pools and tensors made in inference
mode, also rotated in place; memory that caches share with each other or with new rows."""
import pytest
import torch

import flash_attention_v100 as fa
import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def randn(*shape, seed=0, dt=torch.float16):
    return torch.randn(*shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dt).to(DEV)


@pytest.mark.parametrize("grad", [False, True])
def test_pools_of_inference_mode_used_outside_of_it(grad):
    # such pools have no version that autograd could look at: they are written as others are
    L, P, size, Hkv, D, N = 2, 12, 16, 2, 64, 5
    lens, table = [20, 9, 0], [[3, 7, -1], [1, -1, -1], [-1, -1, -1]]
    with torch.inference_mode():
        kc, vc = randn(L, P, size, Hkv, D, seed=1), randn(L, P, size, Hkv, D, seed=2)
        k, v = randn(L, 3, N, Hkv, D, seed=3), randn(L, 3, N, Hkv, D, seed=4)
    assert kc.is_inference()
    with torch.set_grad_enabled(grad):
        want = po.write(kc, vc, k, v, lens, table)
        fa.paged_cache_write_v100(k, v, kc, vc, ints(lens), ints(table))
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
        path = [[1, 4, -1], [0, 2, 3], [0, -1, -1]]
        want = po.accept(kc, vc, lens, path, N, table)
        got = fa.paged_cache_accept_v100(kc, vc, ints(lens), ints(path), N, ints(table))
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and got.tolist() == want[2]
        sources, lens = [0, 0, 1, -1], want[2]
        want = po.fork(kc, vc, table, lens, sources, [2] * 4)
        new, filled = fa.paged_cache_fork_v100(kc, vc, ints(table), ints(lens), ints(sources), 2)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
        assert new.tolist() == want[2] and filled.tolist() == want[3]
        want = po.compact(kc, vc, want[2], want[3])
        new, used = fa.paged_cache_compact_v100(kc, vc, new, filled)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
        assert new.tolist() == want[2] and int(used) == want[3]


def test_rotation_in_place_of_tensors_of_inference_mode():
    table = fa.rotary_table_v100(32, 64)
    with torch.inference_mode():
        q, k = randn(2, 8, 4, 64, seed=5), randn(2, 8, 2, 64, seed=6)
    want = fa.rotary_embedding_v100(q, k, table)
    with torch.no_grad():
        got = fa.rotary_embedding_v100(q, k, table, inplace=True)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_memory_that_is_written_and_read():
    L, P, size, Hkv, D, N = 2, 8, 16, 2, 64, 3
    lens, table = [20, 9], [[3, 7], [1, -1]]
    args = ints(lens), ints(table)
    k, v = randn(2, N, Hkv, D, seed=1), randn(2, N, Hkv, D, seed=2)
    pool = randn(2 * P, size, Hkv, D, seed=3)
    calls = (lambda kc, vc: fa.paged_cache_write_v100(k, v, kc, vc, *args),
             lambda kc, vc: fa.paged_cache_accept_v100(kc, vc, args[0], ints([[1], [0]]), N, args[1]),
             lambda kc, vc: fa.paged_cache_fork_v100(kc, vc, args[1], args[0], ints([0, 0]), 1),
             lambda kc, vc: fa.paged_cache_compact_v100(kc, vc, args[1], args[0]))
    before = pool.clone()
    wide = randn(P, size, Hkv + 1, D, seed=4)
    for call in calls:
        for kc, vc in ((pool[:P], pool[:P]), (pool[:P], pool[P - 1:-1]), (wide[:, :, 1:], wide[:, :, :-1])):
            with pytest.raises(ValueError, match="same memory"):
                call(kc, vc)
    kc, vc = pool[:P], pool[P:]
    for bad in ((kc[:2, :N], v), (k, vc[2:4, 5:5 + N]), (k, kc[-2:, -N:]), (kc[:N, 4:6].transpose(0, 1), v)):
        with pytest.raises(ValueError, match="cache's memory"):
            fa.paged_cache_write_v100(*bad, kc, vc, *args)
    assert torch.equal(pool, before)
    # K and V of a page side by side; a layer's rows from another layer of the same pages
    both = randn(P, 2, L, size, Hkv, D, seed=5)
    kc, vc = both[:, 0, 0], both[:, 1, 0]
    new = both[:2, 0, 1, :N], both[:2, 1, 1, :N]
    rest = both[:, :, 1].clone()
    want = po.write(kc[None], vc[None], new[0][None], new[1][None], lens, table)
    fa.paged_cache_write_v100(*new, kc, vc, *args)
    assert torch.equal(kc, want[0][0]) and torch.equal(vc, want[1][0]) and torch.equal(both[:, :, 1], rest)
