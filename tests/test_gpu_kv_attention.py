"""GPU parity of tq_kv_attention where test_gpu_cache.py does not look: NaN over contexts that are cut into shares,
the bits of 16-bit outputs, and rows that belong to no sequence."""
import math

import numpy as np
import pytest

from test_gpu_cache import CASES, Case, dtype_of, eps_half, least, rand, reference

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


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("new,group", TILES)
@pytest.mark.parametrize("length", [250, 3000])
def test_a_nan_row_that_sees_no_key_is_zeros(tq, codes, new, group, length):
    """Keys without a page are seen by nobody, whatever the row: only such ones, zeros; some such ones among others, what the
    others give (to the rounding of sums in another order), and NaN for the NaN rows."""
    import torch

    c = Case(tq, [length], [new], 16, 2, 64, codes)
    c.fill(9)
    q = rand(10, new, 2 * group, 64)
    q[new // 2, 0, 7], q[new // 3, 1, 8] = math.nan, math.inf
    whole = c.table.clone()
    c.table.fill_(-1)
    assert (c.cache.attention(q, c.batch) == 0).all()
    c.table.copy_(whole)
    c.table[:, :-2:3] = 1 << 20
    got = c.cache.attention(q, c.batch)
    bad = torch.isnan(q).any(-1) | torch.isinf(q).any(-1)
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()


# ------------------------------------------------------------------ the bits of 16-bit outputs
def exact_rows(c, q, b=0):
    """Sequence b's rows in 64 bits on the GPU: (o, sum p |v|, the largest |score| and sum |q k| of each row), [t, h, ...]."""
    import torch

    cache, page, d = c.cache, c.page, c.cache.head_dim
    length, t, heads, group = c.lengths[b], c.new[b], cache.heads, q.shape[1] // cache.heads
    pos = torch.arange(length, device="cuda")
    pages = c.table[b, pos // page].long()

    def floats(codes, scale):
        x = codes[pages, :, pos % page, :d]
        x = x.double() if x.dtype == torch.int8 else x.view(torch.float8_e4m3fn).float().double()
        return (x * scale[pages, :, pos % page].double()[..., None]).transpose(0, 1).contiguous()

    k, v = floats(cache.k, cache.k_scale), floats(cache.v, cache.v_scale)
    rows = slice(int(c.offsets[b]), int(c.offsets[b + 1]))
    qq = q[rows].double().view(t, heads, group, d).transpose(0, 1).reshape(heads, t * group, d)
    s = torch.matmul(qq, k.transpose(1, 2).contiguous()) / math.sqrt(d)
    size = (torch.matmul(qq.abs(), k.abs().transpose(1, 2).contiguous()) / math.sqrt(d)).amax(-1, keepdim=True)
    seen = pos[None] <= (length - t + torch.arange(t, device="cuda"))[:, None]
    s = s.masked_fill(~seen.repeat_interleave(group, 0)[None], -math.inf)
    top = torch.where(s.isinf(), 0.0, s).abs().amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    back = [x.view(heads, t, group, -1).transpose(0, 1).reshape(t, heads * group, -1)
            for x in (torch.matmul(p, v), torch.matmul(p, v.abs()), top, size)]
    return back


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("new,group", TILES)
@pytest.mark.parametrize("length", [8, 200, 777, 4096])
def test_16_bit_outputs_are_the_nearest_ones(tq, codes, dtype, new, group, length):
    """An f32 evaluation gives the 16-bit number nearest to the exact result but where that lies within the evaluation's
    error of a border.  Scores up to 16 with eight f32 roundings are off by 2^-17 relative, one step of the type is eps / 2 to
    eps of the value, and elements smaller than the typical one (their steps are smaller, the errors not) make it
    four times as many: a share of 4 * 2^-17 / eps (f16 3 %, bf16 0.4 %).  Probabilities of 11 bits, off by 2^-12.8 (rms),
    would give 16 and 2 % before that factor."""
    import torch

    if length < new:
        new = length
    dt = dtype_of(dtype)
    c = Case(tq, [length], [new], 64, 8, 128, codes)
    c.fill(7)
    q = rand(8, new, 8 * group, 128, dtype=dt, std=1.5)
    ref = exact_rows(c, q)[0]
    got = c.cache.attention(q, c.batch)
    off = float((got != ref.to(dt)).double().mean())
    assert off <= 4 * 2.0 ** -17 / torch.finfo(dt).eps + 8 / got.numel(), off


def near(got, ref, tol, what=""):
    """`tol` of `reference` (f32 evaluation, in sum p |v| of each element), and one rounding of the element to its type."""
    err = (got.double().cpu() - ref).abs()
    bound = tol + eps_half(got.dtype) * (ref.abs() + tol) + least(got.dtype) + 1e-30
    bad = err > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((err - bound).max()):.3g} over"


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("lengths,new,page,heads,group,d", CASES + [
    ([1500], [100], 64, 1, 2, 128), ([700, 90], [70, 48], 32, 2, 1, 64), ([1000, 20, 400], [33, 20, 5], 16, 1, 2, 96),
    ([400], [129], 16, 1, 1, 33), ([600], [300], 48, 1, 1, 128), ([2000, 1], [9, 1], 16, 1, 5, 80)])
def test_16_bit_attention_by_the_element(tq, codes, dtype, lengths, new, page, heads, group, d):
    """Each element within the bound of its own terms, sum p |v|, not of the cache's largest value."""
    import torch

    c = Case(tq, lengths, new, page, heads, d, codes, seed=d)
    c.fill(15)
    q = rand(16, c.rows, heads * group, d, dtype=dtype_of(dtype), std=1.5)
    seen = torch.rand(c.rows, max(new), generator=torch.Generator().manual_seed(d)) < 0.4
    for tree in (None, seen):
        ref, tol = reference(c, q, tree)
        near(c.cache.attention(q, c.batch, tree=None if tree is None else tq.tree_mask(tree).cuda()), ref, tol,
             f"{lengths} {new} tree={tree is not None}")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("lengths,new,heads,group,d", [
    ([20000, 12345, 300], [40, 33, 40], 4, 1, 64), ([9000, 30000], [3, 1], 4, 4, 128), ([17000], [200], 8, 1, 128),
    ([4000] * 40 + [5], [1] * 41, 4, 2, 32)])
def test_16_bit_attention_of_long_sequences_by_the_element(tq, dtype, lengths, new, heads, group, d):
    """Long sequences, whose outputs are small beside the values: a unit of keys left out would show."""
    c = Case(tq, lengths, new, 64, heads, d, "i8", ragged=True)
    c.fill(33)
    q = rand(34, c.rows, heads * group, d, dtype=dtype_of(dtype), std=1.5)
    got = c.cache.attention(q, c.batch)
    for b in range(len(lengths)):
        ref, pv, top, size = exact_rows(c, q, b)
        tol = 2 * 2.0 ** -24 * ((d + 16) * size + 8 * (top + 64)) * pv
        near(got[int(c.offsets[b]):int(c.offsets[b + 1])], ref.cpu(), tol.cpu(), f"sequence {b}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,group", TILES)
@pytest.mark.parametrize("far", [2, 10, 18, 26, 34])
def test_elements_that_only_light_keys_hold(tq, dtype, new, group, far):
    """One key's values are 2^far times the others' and zero in the last 32 elements: these are the other keys', carried in
    two f16 planes P = hi + lo + e, |e| <= max(2^-22 P, 2^-25), with the row's largest P at 2^8 or more, so off by 2^-22 of
    their terms and 2^-33 of the largest p s for each unit of the codes, next to the f32 evaluation's own bound."""
    import torch

    length, d = 400, 64
    c = Case(tq, [length], [new], 16, 1, d, "i8")
    k, v = rand(61, length, 1, d) * 0.2, rand(62, length, 1, d)
    v[5, :, :32] *= 2.0 ** far
    v[5, :, 32:] = 0.0
    c.cache.write(k, v, c.all_tokens())
    q = rand(63, new, group, d, dtype=dtype_of(dtype))
    ref, pv, top, size = exact_rows(c, q)
    tol = 2 * 2.0 ** -24 * ((d + 16) * size + 8 * (top + 64)) * pv + 2.0 ** -22 * pv
    pos = torch.arange(length, device="cuda")
    at = c.table[0, pos // 16].long()
    codes = c.cache.v[at, 0, pos % 16, :d].double().abs().sum(0)  # of each element
    largest = float(c.cache.v_scale.max())  # p <= 1
    tol = tol + 2.0 ** -33 * largest * codes
    near(c.cache.attention(q, c.batch), ref.cpu(), tol.cpu())
    assert float(c.cache.v_scale.max()) > 2.0 ** (far - 2) * float(c.cache.v_scale[at[6], 0, 6])


# ------------------------------------------------------------------ rows that belong to no sequence
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("most,sequences", [(1, 3), (8, 3), (60, 3), (8, 150)])
@pytest.mark.parametrize("fault", ["long", "past", "before"])
def test_rows_of_no_sequence_are_zeros(tq, dtype, most, sequences, fault):
    """A sequence with more rows than max_tokens, one that reaches past the call's rows, and rows before the first
    sequence: not written to the cache, read as zeros and attended to as zeros, wherever they lie in the batch; the other rows
    as without them."""
    import torch

    dt = dtype_of(dtype)
    new = [most] * sequences
    bad = {"long": sequences // 2, "past": sequences - 1, "before": -1}[fault]
    before = 3 if fault == "before" else 0
    if fault == "long":
        new[bad] = most + 5
    lengths = [100 + i % 7 for i in range(sequences)]
    off = before + np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(off[-1]) - (1 if fault == "past" else 0)
    stray = slice(0, before) if fault == "before" else slice(int(off[bad]), min(int(off[bad + 1]), rows))
    c = Case(tq, lengths, new, 16, 2, 64, "i8")
    c.fill(51)
    kept = [x.clone() for x in (c.cache.k, c.cache.k_scale, c.cache.v, c.cache.v_scale)]
    batch = tq.KVBatch(c.table, c.batch.lengths, most, torch.from_numpy(off.astype(np.int32)).cuda(), rows)
    q, k, v = rand(52, rows, 4, 64, dtype=dt), rand(53, rows, 2, 64, dtype=dt), rand(54, rows, 2, 64, dtype=dt)
    out = torch.full_like(q, 9.0)
    c.cache.attention(q, batch, out=out)
    assert (out[stray] == 0).all()
    for b in {0, sequences // 3, sequences - 2, sequences - 1} - {bad}:
        part = slice(int(off[b]), int(off[b + 1]))
        one = tq.KVBatch(c.table[b:b + 1], c.batch.lengths[b:b + 1], new[b])
        near(out[part], *reference_of(c, q[part], b), f"sequence {b}")
        assert torch.equal(out[part], c.cache.attention(q[part], one)), b  # (one block has each: the same sums)
    back = tuple(torch.full((rows, 2, 64), 5.0, device="cuda") for _ in range(2))
    c.cache.read(batch, torch.float32, back)
    assert all((x[stray] == 0).all() for x in back)
    c.cache.write(k, v, batch)
    if fault != "before":  # the stray sequence's places are as they were
        pages = c.table[bad].long()
        for x, y in zip((c.cache.k, c.cache.k_scale, c.cache.v, c.cache.v_scale), kept):
            assert torch.equal(x[pages], y[pages])
    if before:
        assert torch.equal(c.cache.k[c.table[0].long()][0, :, :50], kept[0][c.table[0].long()][0, :, :50])


def reference_of(c, q, b):
    """Sequence b's rows q in 64 bits, and the bound of `reference`."""
    import torch

    one = Case.__new__(Case)
    one.__dict__.update(c.__dict__)
    one.lengths, one.new = [c.lengths[b]], [q.shape[0]]
    one.table, one.offsets, one.rows = c.table[b:b + 1], np.array([0, q.shape[0]]), q.shape[0]
    return reference(one, q)


@pytest.mark.parametrize("length", [300, 3000])
def test_offsets_that_decrease(tq, length):
    """Nothing is counted twice: sequences of other 64s than that of the decrease are attended to as ever, and so many rows
    counted again that 32 bits would not hold their units are not worked on."""
    import torch

    new = [2] * 200
    c = Case(tq, [length] * 200, new, 16, 2, 64, "i8", ragged=True)
    c.fill(71)
    q = rand(72, 400, 2, 64)
    off = torch.from_numpy(c.offsets).cuda()
    off[70] = 137  # sequence 69 begins at 138
    got = c.cache.attention(q, tq.KVBatch(c.table, c.batch.lengths, 2, off, 400))
    for b in (0, 1, 62, 63, 128, 129, 199):  # (the line of work is another, and so are the shares: not the same bits)
        ref, pv, top, size = exact_rows(c, q, b)
        near(got[2 * b:2 * b + 2], ref.cpu(), (2 * 2.0 ** -24 * (80 * size + 8 * (top + 64)) * pv).cpu(), f"sequence {b}")


def test_offsets_that_decrease_past_32_bits(tq):
    import torch

    rows, heads, page = 1 << 20, 64, 1 << 16
    cache = tq.KVCache.allocate(4, page, heads, 32)
    for sequences in (10, 200):  # five times the rows in one 64, and in several of which some do not decrease
        off = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
        if sequences == 10:
            off[1::2] = rows
        else:
            off[64:] = rows
            off[128] = 0
            off[129:] = rows
        table = torch.arange(4, dtype=torch.int32, device="cuda").expand(sequences, 4).contiguous()
        lengths = torch.full((sequences,), 8, dtype=torch.int32, device="cuda")
        if sequences == 10:
            lengths.fill_(4 * page)
        batch = tq.KVBatch(table, lengths, rows, off, rows)
        q = torch.zeros(rows, heads, 32, dtype=torch.float16, device="cuda")
        out = cache.attention(q, batch)
        torch.cuda.synchronize()
        assert out.shape == q.shape
