"""Outputs of the serving calls that overlap what a call reads, or each other, are refused (CPU: nothing is launched); neighbours
in memory are not (GPU)."""
import pytest

from test_cache_abi import batch, cache, refuse
from test_pages import Pool, at

M = 1 << 20


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def message(abi, what):
    text = abi.lib().tq_last_error().decode()
    assert "overlap" in text, (what, text)


def both_ends(first, size, length):
    """Addresses from which `length` bytes meet the `size` bytes at `first` in their first or in their last element."""
    return first + size - 4, first - length + 4, first


def test_lengths_that_keep_writes(abi):
    """Over a part of the batch's lengths, its table (strided) or offsets, the paths, kept or the cache."""
    n, heads, page, row = 3, 2, 16, 64
    c = cache(abi, k=100 * M, k_scale=110 * M, v=120 * M, v_scale=130 * M)
    b = batch(abi, table=1 * M, table_stride=7, table_pages=2, lengths=2 * M, offsets=3 * M, batch=n, max_tokens=5, tokens=9)
    path, kept = 4 * M, 5 * M
    for first, size in ((1 * M, 4 * (2 * 7 + 2)), (2 * M, 4 * n), (3 * M, 4 * (n + 1)), (path, 4 * (2 * 11 + 6)), (kept, 4 * n),
                        (100 * M, 4 * heads * page * row), (110 * M, 4 * heads * page * 4), (120 * M, 4 * heads * page * row), (130 * M, 4 * heads * page * 4)):
        for out in both_ends(first, size, 4 * n):
            refuse(abi, "tq_kv_keep", at(c), at(b), path, 11, 6, kept, out, None)
            message(abi, (first, out))
