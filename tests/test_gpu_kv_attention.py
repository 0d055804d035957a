"""GPU parity of tq_kv_attention where test_gpu_cache.py does not look: NaN over contexts that are cut into shares,
the bits of 16-bit outputs, and rows that belong to no sequence."""
import math

import numpy as np
import pytest

from test_gpu_cache import Case, dtype_of, rand

pytestmark = pytest.mark.gpu

# new tokens, group: tiles of 16, 32, 64 and 128 rows
TILES = [(1, 4), (20, 1), (50, 1), (200, 1)]


# ------------------------------------------------------------------ NaN in what a row sees
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,group", TILES)
@pytest.mark.parametrize("length,heads", [(300, 2), (3000, 2), (30000, 1), (3000, 40)])
def test_a_nan_row_is_nan_however_its_keys_are_cut(tq, dtype, new, group, length, heads):
    """A NaN in a row of q makes all of its scores NaN, whether one block works on its keys, a few or very many; the other
    rows keep their bits.  An infinity does the same (its products with keys of both signs)."""
    import torch

    c = Case(tq, [length], [new], 64, heads, 64, "i8")
    c.fill(3)
    q = rand(4, new, heads * group, 64, dtype=dtype_of(dtype))
    want = c.cache.attention(q, c.batch)
    for bad in (math.nan, math.inf):
        x = q.clone()
        row, head = new // 2, heads * group - 1
        x[row, head, 5] = bad
        got = c.cache.attention(x, c.batch)
        assert torch.isnan(got[row, head]).all(), (bad, got[row, head, :4])
        got[row, head] = want[row, head]
        assert torch.equal(got, want), bad


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("new,group", TILES)
@pytest.mark.parametrize("units,heads", [(3, 2), (24, 2), (200, 1), (24, 40)])
def test_a_nan_key_alone_in_its_share_reaches_the_rows(tq, codes, new, group, units, heads):
    """The newest key, the first of its 128, has an infinite scale (0 * inf): the last row sees it, and no other."""
    import torch

    length = 128 * units + 1
    c = Case(tq, [length], [new], 64, heads, 64, codes)
    k, v = c.fill(5)
    q = rand(6, new, heads * group, 64)
    want = c.cache.attention(q, c.batch)
    k[-1, :, 3] = math.inf
    c.cache.write(k, v, c.all_tokens())
    got = c.cache.attention(q, c.batch)
    assert torch.isnan(got[-1]).all()
    assert torch.equal(got[:-1], want[:-1]) and torch.isfinite(want).all()
