"""The paged cache at its edges, on a machine without a GPU: the largest writes."""
from test_paged_cpu import CODES, status, write_args


def test_largest_writes():
    # 4 rows of each of 4 waves a workgroup: fewer than 2^24 workgroups of 256 threads
    for rows, code in (((1 << 28) - 16, "FA_OK"), ((1 << 28) - 15, "FA_ERR_TOO_LARGE"), ((1 << 28) - 1, "FA_ERR_TOO_LARGE")):
        a = write_args(N=1, batch=1)
        a.tokens = rows
        assert status("fa_cache_write", a) == CODES[code], rows
    a = write_args(N=(1 << 14) - 1, batch=1 << 14)
    assert status("fa_cache_write", a) == CODES["FA_OK"]
