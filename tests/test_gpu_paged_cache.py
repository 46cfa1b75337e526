"""Operators of the paged cache against lists: writes, accepted drafts, forks,
compaction; whole pools are compared, so that nothing else is written."""
import pytest
import torch

import flash_attention_v100 as fa
import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def ints(x, dtype=torch.int32):
    return None if x is None else torch.tensor(x, dtype=dtype, device=DEV)


def pools(L, P, size, Hkv, D, dt, seed=0):
    g = torch.Generator("cpu").manual_seed(seed)
    return tuple(torch.randn(L, P, size, Hkv, D, generator=g).to(DT[dt]).to(DEV) for _ in range(2))


def same(got, want):
    for g, w in zip(got, want):
        if isinstance(w, torch.Tensor):
            assert torch.equal(g, w)
        else:
            assert g.dtype == torch.int32 and g.tolist() == w


@pytest.mark.parametrize("dt,Hkv,D", [("bf16", 8, 128), ("fp16", 3, 80), ("fp32", 1, 36), ("bf16", 1, 8), ("fp32", 16, 128)])
@pytest.mark.parametrize("N", [1, 5, 130])
def test_write(dt, Hkv, D, N):
    rng = po.rng(dt, N)
    lens = [N, N + 7, 0, N - 1, N + 40, 300]
    M, P = 20, 60
    kc, vc = pools(1, P, 16, Hkv, D, dt, seed=N)
    table = po.draw_table(rng, lens, 16, M, P)
    k, v = pools(1, 6, N, Hkv, D, dt, seed=N + 1)
    want = po.write(kc, vc, k, v, lens, table)
    got = fa.paged_cache_write_v100(k[0], v[0], kc[0], vc[0], ints(lens), ints(table))
    assert got[0].data_ptr() == kc.data_ptr() and got[1].data_ptr() == vc.data_ptr()
    same((kc, vc), want)


@pytest.mark.parametrize("L,N", [(3, 2), (40, 1), (5, 700)])
def test_write_layers(L, N):
    lens = [N + 3, N, 0]
    table = po.draw_table(po.rng(L), lens, 32, 24, 60)
    kc, vc = pools(L, 60, 32, 2, 64, "bf16")
    k, v = pools(L, 3, N, 2, 64, "bf16", seed=1)
    want = po.write(kc, vc, k, v, lens, table)
    fa.paged_cache_write_v100(k, v, kc, vc, ints(lens), ints(table))
    same((kc, vc), want)


@pytest.mark.parametrize("dt,Hkv,D", [("fp16", 1, 8), ("fp32", 1, 36), ("bf16", 3, 80), ("bf16", 1, 128), ("fp16", 4, 64)])
def test_write_many_short_rows(dt, Hkv, D):
    # rows of 1, 9, 30, 16 and 32 chunks, several rows a wave (64, 7, 2, 4, 2), heads apart in the pool
    L, N, lens = 2, 5500, [5500, 3000, 5511]
    table = po.draw_table(po.rng(dt, D), lens, 32, 173, 460)
    kc, vc = pools(L, 460, 32, Hkv, D, dt)
    vc = vc.transpose(2, 3).contiguous().transpose(2, 3)
    k, v = pools(L, 3, N, Hkv, D, dt, seed=1)
    want = po.write(kc, vc, k, v, lens, table)
    fa.paged_cache_write_v100(k, v, kc, vc, ints(lens), ints(table))
    same((kc, vc), want)


def test_write_rows_strides_and_no_pages():
    # rows of tokens; strided inputs and pools; pages that are none; lengths past the room
    kc, vc = pools(1, 3, 50, 2, 64, "fp16")
    k, v = pools(1, 3, 4, 2, 64, "fp16", seed=2)
    lens = [50, 4, 2]
    want = po.write(kc, vc, k, v, lens, None)
    wide = torch.cat([k[0], k[0]], -1)[..., :64]
    pool = vc[0].transpose(0, 1).contiguous().transpose(0, 1)
    fa.paged_cache_write_v100(wide, v[0].transpose(1, 2).contiguous().transpose(1, 2), kc[0], pool, ints(lens))
    same((kc[0], pool), (want[0][0], want[1][0]))
    fa.paged_cache_write_v100(k[0], v[0], kc[0], vc[0], ints([51, 2 ** 31 - 1, -3]))
    want = po.write(kc, vc, k, v, [50, 50, -3], None)
    same((kc, vc), want)
    kc, vc = pools(1, 5, 16, 2, 64, "fp16")
    k, v = pools(1, 2, 40, 2, 64, "fp16", seed=3)
    table = [[0, -1, 3], [5, 2 ** 31 - 1, 1]]
    want = po.write(kc, vc, k, v, [48, 41], table)
    fa.paged_cache_write_v100(k[0], v[0], kc[0], vc[0], ints([48, 41]), ints(table))
    same((kc, vc), want)


@pytest.mark.parametrize("dt,Hkv,D", [("bf16", 8, 128), ("fp16", 3, 80), ("fp32", 1, 36)])
@pytest.mark.parametrize("N", [1, 9, 64, 200])
def test_accept(dt, Hkv, D, N):
    rng = po.rng("accept", N)
    B, A = 12, min(N, 20)
    lens = [N + rng.randint(0, 40) for _ in range(B)]
    lens[3], lens[5] = N - 1, 0
    path = [sorted(rng.sample(range(N), rng.randint(0, A))) for _ in range(B)]
    path = [p + [-1] * (A - len(p)) for p in path]
    path[0] = list(range(A))                    # nothing moves
    path[1] = list(range(N - A, N))             # all from the end
    path[2] = [0, 0] + [1] * (A - 2) if A >= 2 else [N]
    M = -(-(N + 40) // 16)
    P = B * M + 1
    table = po.draw_table(rng, lens, 16, M, P)
    kc, vc = pools(2, P, 16, Hkv, D, dt, seed=N)
    want = po.accept(kc, vc, lens, path, N, table)
    got = fa.paged_cache_accept_v100(kc, vc, ints(lens), ints(path), N, ints(table))
    same((kc, vc, got), want)


def test_accept_long_paths_rows_and_what_is_none():
    N, room = 150, 170
    kc, vc = pools(1, 4, room, 2, 64, "bf16")
    path = [list(range(1, 141)), list(range(10, 150)), [2 ** 31 - 1] + [0] * 139, list(range(0, 128)) + [5] * 12]
    lens = [170, 150, 160, 155]
    want = po.accept(kc, vc, lens, path, N, None)
    got = fa.paged_cache_accept_v100(kc[0], vc[0], ints(lens, torch.int64), ints(path, torch.int64), N)
    same((kc, vc, got), want)
    kc, vc = pools(1, 6, 16, 2, 64, "bf16")
    table = [[0, -1, 4], [1, 2, 6]]
    path = [[0, 14, 31], [1, 20, 40]]
    want = po.accept(kc, vc, [40, 48], path, 42, table)
    got = fa.paged_cache_accept_v100(kc[0], vc[0], ints([40, 48]), ints(path), 42, ints(table))
    same((kc, vc, got), want)
    assert fa.paged_cache_accept_v100(kc[0], vc[0], ints([40, 48]), ints([[], []]), 3, ints(table)).tolist() == [37, 45]


def random_fork(seed, B, Bn, M, P, size, L, more_max, shared=True):
    rng = po.rng("fork", seed)
    lens, table, pages = [], [], list(range(P))
    rng.shuffle(pages)
    for _ in range(B):
        n = min(rng.randint(0, M * size), max(0, len(pages) - 2) * size)
        k = -(-n // size)
        lens.append(n)
        table.append([pages.pop() for _ in range(k)] + [rng.choice([-1, 0, P, 1]) for _ in range(M - k)])
    if shared and B > 2:  # whole pages that two sequences share
        k = min(lens[0], lens[1]) // size // 2
        table[1][:k] = table[0][:k]
    sources = [rng.choice([-1, B, *range(B), *range(B)]) for _ in range(Bn)]
    more = [rng.randint(-1, more_max) for _ in range(Bn)]
    return lens, table, sources, more


@pytest.mark.parametrize("seed", range(12))
def test_fork(seed):
    B, Bn, M, P, size, L = [(5, 7, 6, 60, 16, 2), (1, 9, 3, 40, 32, 1), (40, 40, 5, 260, 16, 1), (3, 0, 2, 8, 16, 1),
                            (8, 30, 9, 90, 16, 3), (6, 6, 4, 16, 48, 1)][seed % 6]
    lens, table, sources, more = random_fork(seed, B, Bn, M, P, size, L, 40)
    kc, vc = pools(L, P, size, 2, 64, "bf16", seed=seed)
    want = po.fork(kc, vc, table, lens, sources, more)
    dt = torch.int64 if seed % 2 else torch.int32
    got = fa.paged_cache_fork_v100(kc, vc, ints(table, dt), ints(lens, dt), ints(sources, dt).flatten(), ints(more, dt).flatten())
    same((kc, vc, got[0], got[1]), (*want[:2], want[2] if Bn else [], want[3]))


@pytest.mark.parametrize("dt,Hkv,D,size", [("fp32", 5, 100, 16), ("fp16", 8, 128, 256), ("bf16", 1, 8, 16)])
def test_fork_types(dt, Hkv, D, size):
    lens = [3 * size - 1, size + 1, 0]
    table = [[7, 2, 9], [4, 0, -1], [-1] * 3]
    kc, vc = pools(2, 12, size, Hkv, D, dt)
    sources = [0, 0, 1, 0, 1, 2]
    want = po.fork(kc, vc, table, lens, sources, [1] * 6)
    got = fa.paged_cache_fork_v100(kc, vc, ints(table), ints(lens), ints(sources), 1)
    same((kc, vc, *got), want)


def test_fork_that_runs_out():
    # in the batch's order, until the first that finds no page; no room in the table
    lens, table = [40, 16, 5], [[0, 1, 2], [3, -1, -1], [4, -1, -1]]
    for P in (5, 6, 7, 8, 9, 20):
        kc, vc = pools(1, P, 16, 1, 8, "bf16", seed=P)
        sources, more = [0, 0, 1, 1, 2, 2, 0], [8, 8, 0, 1, 11, 0, 9]
        want = po.fork(kc, vc, table, lens, sources, more)
        got = fa.paged_cache_fork_v100(kc[0], vc[0], ints(table), ints(lens), ints(sources), ints(more))
        same((kc, vc, *got), want)


def test_fork_of_pages_that_are_none():
    lens, table = [40, 40], [[0, -1, 2], [1, 3, 99]]
    kc, vc = pools(1, 8, 16, 1, 8, "bf16")
    sources, more = [1, 1, 0, 1, 0], [0] * 5
    want = po.fork(kc, vc, table, lens, sources, more)
    got = fa.paged_cache_fork_v100(kc[0], vc[0], ints(table), ints(lens), ints(sources))
    same((kc, vc, *got), want)


def test_fork_and_compact_large_pools():
    # the form for more than 2^17 pages, lengths past the room
    P, M = (1 << 17) + 77, 9
    kc = torch.arange(P * 16, device=DEV, dtype=torch.float32).view(1, P, 16, 1, 1).expand(1, P, 16, 1, 8).contiguous()
    kc, vc = kc, kc + 0.5
    rng = po.rng("large")
    lens = [rng.randint(0, M * 16) for _ in range(50)] + [10 ** 6]
    table = [[rng.randrange(P // 2, P) if b % 2 else rng.randrange(P) for _ in range(M)] for b in range(51)]
    pages = iter(rng.sample(range(P), 51 * M))
    table = [[next(pages) for _ in r] for r in table]
    sources = [rng.randrange(51) for _ in range(1500)]
    want = po.fork(kc, vc, table, lens, sources, [20] * 1500)
    got = fa.paged_cache_fork_v100(kc, vc, ints(table), ints(lens), ints(sources), 20)
    same((kc, vc, *got), want)
    want = po.compact(kc, vc, got[0].tolist(), got[1].tolist())
    got = fa.paged_cache_compact_v100(kc, vc, *got)
    same((kc, vc, *got), want)


@pytest.mark.parametrize("B,Bn,P", [(1100, 1500, 6000), (1100, 70, 3000), (60, 1500, 9000)])
def test_batches_of_more_than_a_workgroup(B, Bn, P):
    lens, table, sources, more = random_fork(B + Bn, B, Bn, 3, P, 16, 1, 20)
    kc, vc = pools(1, P, 16, 1, 8, "bf16", seed=Bn)
    want = po.fork(kc, vc, table, lens, sources, more)
    got = fa.paged_cache_fork_v100(kc, vc, ints(table), ints(lens), ints(sources), ints(more))
    same((kc, vc, *got), want)
    want = po.compact(kc, vc, got[0].tolist(), got[1].tolist())
    got = fa.paged_cache_compact_v100(kc, vc, *got)
    same((kc, vc, *got), want)


@pytest.mark.parametrize("seed", range(8))
def test_compact(seed):
    B, M, P, size, L = [(5, 6, 60, 16, 2), (1, 3, 40, 32, 1), (40, 5, 260, 16, 3), (3, 2, 6, 48, 1)][seed % 4]
    lens, table, _, _ = random_fork(seed, B, 1, M, P, size, L, 0)
    kc, vc = pools(L, P, size, 3, 40, "fp16", seed=seed)
    want = po.compact(kc, vc, table, lens)
    got = fa.paged_cache_compact_v100(kc, vc, ints(table), ints(lens))
    assert got[1].shape == ()
    same((kc, vc, *got), want)
    again = fa.paged_cache_compact_v100(kc, vc, *[got[0], ints(lens)])
    same((kc, vc, *again), (want[0], want[1], want[2], want[3]))


def test_compact_of_nothing_and_of_all():
    kc, vc = pools(1, 4, 16, 1, 8, "bf16")
    before = kc.clone()
    table, used = fa.paged_cache_compact_v100(kc, vc, ints([[3, 2], [1, 0]]), ints([0, 0]))
    assert table.tolist() == [[-1, -1], [-1, -1]] and int(used) == 0 and torch.equal(kc, before)
    table, used = fa.paged_cache_compact_v100(kc, vc, ints([[3, 2], [1, 0]]), None)
    assert table.tolist() == [[3, 2], [1, 0]] and int(used) == 4 and torch.equal(kc, before)
    table, used = fa.paged_cache_compact_v100(kc, vc, ints([[3, 9], [-1, 3]]), ints([32, 17]))
    assert table.tolist() == [[0, -1], [-1, 0]] and int(used) == 1 and torch.equal(kc[:, 0], before[:, 3])


def test_empty_batches():
    kc, vc = pools(1, 4, 16, 1, 8, "bf16")
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    t = torch.empty(0, 3, dtype=torch.int32, device=DEV)
    assert fa.paged_cache_compact_v100(kc, vc, t, e)[1].item() == 0
    assert fa.paged_cache_fork_v100(kc, vc, t, e, ints([0, -1]), 2)[1].tolist() == [0, 0]
    assert fa.paged_cache_accept_v100(kc, vc, e, t, 3, t).shape == (0,)
    k = kc[:, :0, :2]
    fa.paged_cache_write_v100(k, k, kc, vc, e, t)
    table, lens = fa.paged_cache_fork_v100(kc, vc, ints([[1, 2]]), ints([20]), ints([0]), 0)
    assert table.tolist() == [[1, 2]] and lens.tolist() == [20]
