"""The paged cache at its edges, on a machine without a GPU: the largest writes, tensors that
share memory."""
import random

import torch

from flash_attention_v100 import _paged
from test_paged_cpu import CODES, status, write_args


def test_largest_writes():
    # 4 rows of each of 4 waves a workgroup: fewer than 2^24 workgroups of 256 threads
    for rows, code in (((1 << 28) - 16, "FA_OK"), ((1 << 28) - 15, "FA_ERR_TOO_LARGE"), ((1 << 28) - 1, "FA_ERR_TOO_LARGE")):
        a = write_args(N=1, batch=1)
        a.tokens = rows
        assert status("fa_cache_write", a) == CODES[code], rows
    a = write_args(N=(1 << 14) - 1, batch=1 << 14)
    assert status("fa_cache_write", a) == CODES["FA_OK"]


def elements(t):
    out = {t.data_ptr()}
    for n, st in zip(t.shape, t.stride()):
        out = {x + i * st * t.element_size() for x in out for i in range(n)}
    return out if t.numel() else set()


def test_shared_memory_against_all_elements():
    rng, shares = random.Random(1), _paged.host().shares
    seen = [0, 0]
    for _ in range(4000):
        buf = torch.empty(rng.randint(60, 400))
        views = []
        for _ in range(2):
            shape = [rng.choice([1, 1, 2, 3, 4]) for _ in range(rng.randint(1, 4))]
            strides = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48]) for _ in shape]
            room = buf.numel() - 1 - sum((n - 1) * st for n, st in zip(shape, strides))
            views.append(buf.as_strided(shape, strides, rng.randint(0, room)) if room >= 0 else buf[:0])
        want = bool(elements(views[0]) & elements(views[1]))
        assert shares(*views) == want == shares(*views[::-1]), [(v.shape, v.stride(), v.storage_offset()) for v in views]
        seen[want] += 1
    assert min(seen) > 100


def test_shared_memory_of_large_pools():
    # K and V of a page, layers, heads side by side; exact however many pages there are
    shares = _paged.host().shares
    pool = torch.empty(3000, 2, 16, 2, 16, dtype=torch.float16)
    k, v = pool[:, 0], pool[:, 1]
    assert not shares(k, v) and not shares(v, k) and shares(k, k) and shares(k, pool) and shares(v[5:6, 3:4], v)
    assert not shares(pool[..., 0, :], pool[..., 1, :]) and shares(pool[1000:], pool[:1001]) and not shares(pool[1000:], pool[:1000])
    rows = torch.empty(2, 3000, 16, 2, 16, dtype=torch.float16)
    assert not shares(rows[0], rows[1]) and shares(rows[0, :7].transpose(0, 1), rows)
    assert not shares(pool[:, 0, :, 0], pool.transpose(1, 2)[:, :, 0, 1]) and shares(pool[:, 0, :, 0], pool.transpose(1, 2)[:, 3])
    assert not shares(torch.empty(0), pool) and not shares(pool, torch.empty(3))
