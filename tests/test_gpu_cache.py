"""GPU parity: rotary positions, the 8-bit key/value cache and attention over it
(tq_rotary_apply, tq_kv_write[_rotary], tq_kv_read, tq_kv_attention) against plain 64-bit
computations, at the sizes, masks, strides and descriptors where they can go wrong."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


def eps_half(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half a step of the type's subnormals, whose rounding is absolute (f16: 2^-25)."""
    import torch

    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def rand(seed, *shape, dtype=None, std=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype or torch.float32)


def dtype_of(name):
    import torch

    return getattr(torch, name)


# ------------------------------------------------------------------ rotary
def turned(x, pos, f, m, pairs, inverse=False):
    """x [n, h, d] by exact angles, and what each element's error may be: 6 roundings of f32
    in cosine or sine (polynomial 2, scale 1), product and sum, then one to the type."""
    x, f = x.double().cpu(), f.double().cpu()
    a = pos.double().cpu()[:, None] * f
    a = -a if inverse else a
    c, s = (a.cos() * m)[:, None], (a.sin() * m)[:, None]
    r = 2 * f.numel()
    y, size = x.clone(), x.abs()
    i0, i1 = (slice(0, r, 2), slice(1, r, 2)) if pairs else (slice(0, r // 2), slice(r // 2, r))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    both = (x[..., i0].abs() + x[..., i1].abs()) * m
    size[..., i0] = both
    size[..., i1] = both
    return y, size * 6 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,h,hk,d,r,pairs", [
    (1, 1, 1, 128, 128, False), (3, 4, 2, 128, 64, True), (65, 8, 8, 64, 64, False), (7, 5, 1, 80, 80, False),
    (5, 3, 3, 80, 40, True), (2, 2, 1, 5, 4, False), (9, 2, 2, 96, 48, False), (4, 3, 1, 100, 50, True),
    (1100, 6, 2, 32, 16, False), (2, 1, 0, 1, 0, False), (3, 2, 2, 128, 18, False), (6, 2, 2, 128, 2, True)])
def test_rotary(tq, dtype, n, h, hk, d, r, pairs):
    import torch

    dt = dtype_of(dtype)
    q, k = rand(n + d, n, h, d, dtype=dt), rand(n + d + 1, n, hk, d, dtype=dt) if hk else None
    rot = tq.Rotary.from_base(r, 10000.0, pairs, scale=1.25)
    pos = torch.randint(0, 1 << 20, (n,), generator=torch.Generator().manual_seed(d)).cuda()
    for inverse in (False, True):
        got = rot.apply(q, k, pos, inverse=inverse)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            ref, tol = turned(x, pos, rot.frequencies, 1.25, pairs, inverse)
            err = (y.double().cpu() - ref).abs()
            assert y.dtype == dt and y.shape == x.shape
            assert (err <= tol + eps_half(dt) * ref.abs() * (1 + 2.0 ** -20) + least(dt)).all(), float((err - tol).max())
            assert torch.equal(y[..., r:], x[..., r:])


def test_rotary_reads_slices_of_a_projection_and_gives_the_gradient(tq):
    import torch

    n, h, d = 33, 4, 64
    qkv = rand(5, n, 3 * h * d)
    q, k = qkv[:, :h * d].view(n, h, d), qkv[:, h * d:2 * h * d].view(n, h, d)
    assert not q.is_contiguous()
    rot = tq.Rotary.from_base(d, scaling="linear", factor=4.0)
    pos = torch.arange(n, device="cuda") * 1000
    a, b = rot.apply(q, k, pos)
    c, e = rot.apply(q.contiguous(), k.contiguous(), pos)
    assert torch.equal(a, c) and torch.equal(b, e)
    # the gradient of sum(w * turned(q)) is w turned back: against differences in 64 bits, in which
    # the operator is linear, so that a step of 1 is exact
    w = rand(6, n, h, d)
    got = rot.apply(w, None, pos, inverse=True)[0].double().cpu()
    for i in (0, 17, 31, 32, 63):
        step = torch.zeros(n, h, d, dtype=torch.float64)
        step[..., i] = 1.0
        moved, _ = turned(step, pos, rot.frequencies, 1.0, False)
        assert ((w.double().cpu() * moved).sum(-1) - got[..., i]).abs().max() < 6 * 2.0 ** -24 * 2 * float(w.abs().max())
    # a strided head dimension and odd strides take the element path: the same numbers
    wide = rand(7, n, h, 2 * d)[..., ::2]
    assert torch.equal(rot.apply(wide, None, pos)[0], rot.apply(wide.contiguous(), None, pos)[0])
    odd = rand(8, n * (h * d + 1) + 8)[:n * (h * d + 1)].view(n, -1)[:, 1:].view(n, h, d)
    assert torch.equal(rot.apply(odd, None, pos)[0], rot.apply(odd.contiguous(), None, pos)[0])


# ------------------------------------------------------------------ cache
class Case:
    """A batch of sequences on shuffled pages, and the plain view of what lies where."""

    def __init__(self, tq, lengths, new, page, heads, d, codes, ragged=False, spare=2, seed=0, extra=0):
        import torch

        self.tq, self.lengths, self.new, self.page = tq, lengths, new, page
        per = max(1, max((n + page - 1) // page for n in lengths))
        pages = len(lengths) * per + spare
        order = np.random.default_rng(seed).permutation(pages)[:len(lengths) * per].reshape(len(lengths), per)
        self.table = torch.from_numpy(order.astype(np.int32)).cuda()
        self.cache = tq.KVCache.allocate(pages, page, heads, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + extra
        if ragged or extra or len(set(new)) > 1:
            self.batch = tq.KVBatch(self.table, torch.tensor(lengths, dtype=torch.int32).cuda(), max(new),
                                    torch.from_numpy(self.offsets).cuda(), self.rows)
        else:
            self.batch = tq.KVBatch(self.table, torch.tensor(lengths, dtype=torch.int32).cuda(), new[0])

    def all_tokens(self):
        """A batch that covers every token of every sequence."""
        import torch

        off = np.concatenate([[0], np.cumsum(self.lengths)]).astype(np.int32)
        return self.tq.KVBatch(self.table, self.batch.lengths, max(max(self.lengths), 1), torch.from_numpy(off).cuda(),
                               int(off[-1]))

    def fill(self, seed, std=1.0, dtype=None):
        """Every token written; returns k, v [tokens of all sequences, heads, d]."""
        import torch

        b = self.all_tokens()
        shape = (b.rows, self.cache.heads, self.cache.head_dim)
        k = rand(seed, *shape, std=std, dtype=dtype)
        grow = torch.linspace(0.5, 1.5, b.rows, device="cuda").view(-1, 1, 1)
        v = (rand(seed + 1, *shape, std=std) * grow).to(dtype or torch.float32)
        self.cache.write(k, v, b)
        return k, v


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new,page,heads,d", [
    ([1], [1], 16, 1, 128), ([5, 40, 1], [1, 1, 1], 16, 3, 128), ([33, 47], [33, 20], 32, 2, 80),
    ([64, 17, 0, 3], [7, 17, 0, 2], 48, 2, 64), ([129], [129], 128, 4, 5), ([20, 20], [3, 3], 16, 2, 100),
    ([1500], [1400], 64, 2, 96)])
def test_cache_codes_are_the_row_formats(tq, codes, dtype, lengths, new, page, heads, d):
    """Codes and scales bit for bit those of quantize_per_channel_* on the heads as rows, in the places the table
    names; nothing else is touched; read gives f32(code * scale) rounded once."""
    import torch

    dt = dtype_of(dtype)
    c = Case(tq, lengths, new, page, heads, d, codes)
    cache, n = c.cache, c.rows
    for t in (cache.k, cache.v):
        t.fill_(77)
    cache.k_scale.fill_(-3.0)
    k, v = rand(1, n, heads, d, dtype=dt), rand(2, n, heads, d, dtype=dt)
    k[0, 0, 0] = float("nan")
    v[n - 1, heads - 1, :] = 0.0
    k[n - 1, 0, d - 1] = float("inf") if d > 1 else 1.0
    cache.write(k, v, c.batch)
    quant = tq.quantize_per_channel_i8 if codes == "i8" else tq.quantize_per_channel_fp8
    untouched = torch.ones(cache.k.shape[:3], dtype=torch.bool)
    row = 0
    for x, cc, cs in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        q, s = quant(x.float().reshape(n * heads, d).contiguous())
        q, s = q.view(n, heads, d).cpu(), s.view(n, heads).cpu()
        hc, hs = cc.cpu(), cs.cpu()
        row = 0
        for b, (length, t) in enumerate(zip(lengths, new)):
            for i in range(t):
                p = length - t + i
                page_no, off = int(c.table[b, p // page]), p % page
                assert torch.equal(hc[page_no, :, off, :d], q[row]) and torch.equal(hs[page_no, :, off], s[row])
                assert (hc[page_no, :, off, d:] == 0).all()
                untouched[page_no, :, off] = False
                row += 1
        assert (hc[untouched] == 77).all()
    assert row == n and (cache.k_scale.cpu()[untouched] == -3.0).all()
    deq = tq.dequantize_per_channel_i8 if codes == "i8" else tq.dequantize_per_channel_fp8
    for out in (torch.float32, dt):
        back = cache.read(c.batch, out)
        for x, y in zip((k, v), back):
            q, s = quant(x.float().reshape(n * heads, d).contiguous())
            ref = deq(q, s).view(n, heads, d).to(out)
            assert y.dtype == out and torch.equal(torch.isnan(y), torch.isnan(ref))
            assert torch.equal(torch.nan_to_num(y.float()), torch.nan_to_num(ref.float()))


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,r,pairs,h,hk", [(128, 128, False, 8, 2), (64, 32, True, 3, 3), (80, 80, False, 4, 1), (6, 4, False, 2, 2),
                                            (96, 96, True, 2, 2)])
def test_write_rotary_is_rotary_then_write(tq, codes, dtype, d, r, pairs, h, hk):
    import torch

    dt = dtype_of(dtype)
    lengths, new = [40, 9, 70], [5, 9, 1]
    a, b = (Case(tq, lengths, new, 16, hk, d, codes) for _ in range(2))
    n = a.rows
    # one buffer for the three, as a fused projection leaves them
    buf = rand(3, n, (h + 2 * hk) * d, dtype=dt)
    q, k, v = (x.view(n, -1, d) for x in (buf[:, :h * d], buf[:, h * d:(h + hk) * d], buf[:, (h + hk) * d:]))
    rot = tq.Rotary.from_base(r, 1000.0, pairs, scale=0.75)
    place = torch.tensor([x for l, t in zip(lengths, new) for x in range(l - t, l)]).cuda()
    for positions in (None, place * 100 + 7):
        got = a.cache.write_rotary(q, k, v, rot, a.batch, positions)
        at = place if positions is None else positions
        assert torch.equal(got, rot.apply(q, None, at)[0])
        b.cache.write(rot.apply(k.float(), None, at)[0], v.float(), b.batch)
        for name in ("k", "k_scale", "v", "v_scale"):
            assert torch.equal(getattr(a.cache, name), getattr(b.cache, name)), name


def test_rows_without_a_place(tq):
    """Bad pages, lengths past the table and before their new tokens, rows behind the last sequence:
    not written, read as zeros, left as they were."""
    import torch

    page, heads, d = 16, 2, 64
    cache = tq.KVCache.allocate(4, page, heads, d)
    table = torch.tensor([[0, 9], [-1, 1], [2, 3], [2, 3]], dtype=torch.int32).cuda()
    lengths = torch.tensor([18, 18, 40, 2], dtype=torch.int32).cuda()   # 40 > 32; 2 < 4 new ones
    new = [4, 4, 4, 4]
    off = torch.tensor([0, 4, 8, 12, 16], dtype=torch.int32).cuda()
    batch = tq.KVBatch(table, lengths, 4, off, 19)
    k, v = rand(1, 19, heads, d), rand(2, 19, heads, d)
    cache.write(k, v, batch)
    # sequence 0: positions 14, 15 on page 0, 16, 17 on page 9 (none); 1: 14, 15 on page -1, 16, 17 on 1;
    # 2: 36.. past the table; 3: positions -2, -1, 0, 1 -> the last two on page 2
    lies = [0, 1, 6, 7, 14, 15]
    out = tuple(torch.full((19, heads, d), 5.0, device="cuda") for _ in range(2))
    cache.read(batch, torch.float32, out)
    for x, y in zip((k, v), out):
        ref = tq.fake_quantize_per_channel_i8(x.reshape(-1, d))[2].view(19, heads, d)
        for row in range(19):
            if row >= 16:
                assert (y[row] == 5.0).all(), row
            elif row in lies:
                assert torch.equal(y[row], ref[row]), row
            else:
                assert (y[row] == 0).all(), row
    assert int((cache.k_scale != 0).sum()) == len(lies) * heads
    q = rand(3, 19, 4, d)
    o = torch.full_like(q, 7.0)
    cache.attention(q, batch, out=o)
    assert (o[16:] == 7.0).all() and torch.isfinite(o).all()
    assert (o[12:14] == 0).all()  # before position 0: nothing to see
    assert sum(new) == 16


# ------------------------------------------------------------------ attention
def reference(c, q, tree=None, scale=None):
    """Softmax attention of the batch's rows in 64 bits over what the cache holds, and what an
    f32 evaluation may be off by: a score is off by (d + 16) f32 roundings of its absolute products
    (accumulation, two planes of q of 22 bits), its exponent and the scale's logarithm by 8 more of
    its size; the output by twice the largest of these times sum p |v|."""
    import torch

    cache, d, page = c.cache, c.cache.head_dim, c.page
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    h, hk = q.shape[1], cache.heads
    g = h // hk

    def floats(x):
        x = x.cpu()
        return x.double() if x.dtype == torch.int8 else x.view(torch.float8_e4m3fn).to(torch.float32).double()

    kk, vv = (floats(x)[..., :d] * s.cpu().double()[..., None] for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    out, tol = torch.zeros(c.rows, h, d, dtype=torch.float64), torch.zeros(c.rows, h, d, dtype=torch.float64)
    table = c.table.cpu().long()
    for b, (length, t_new) in enumerate(zip(c.lengths, c.new)):
        first = int(c.offsets[b])
        pos = torch.arange(length)
        pages = table[b, pos // page]
        k, v = kk[pages, :, pos % page], vv[pages, :, pos % page]  # [length, hk, d]
        for t in range(t_new):
            row = first + t
            see = pos <= length - t_new + t
            if tree is not None:
                j = pos - (length - t_new)
                see = torch.tensor([bool(x < 0) or bool(tree[row][x]) for x in j.tolist()], dtype=torch.bool)
            if not see.any():
                continue
            for x in range(h):
                kx, vx, qx = k[see, x // g], v[see, x // g], q[row, x].double().cpu()
                s = kx @ qx * scale
                size = (kx.abs() @ qx.abs()) * abs(scale)
                p = torch.softmax(s, -1)
                out[row, x] = p @ vx
                off = 2.0 ** -24 * ((d + 16) * size.max() + 8 * (s.abs().max() + 64))
                tol[row, x] = 2 * off * (p @ vx.abs())
    return out, tol


def check(got, ref, tol, what=""):
    import torch

    dt = got.dtype
    err = (got.double().cpu() - ref).abs()
    bound = tol + (eps_half(dt) * ref.abs() if dt != torch.float32 else 2.0 ** -22 * ref.abs())
    if dt != torch.float32:  # probabilities rounded to f16 once: half a step of each term
        bound = bound + tol.new_tensor(2.0 ** -11) * p_abs(tol)
    bad = err > bound + least(dt) + 1e-30
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((err - bound).max()):.3g} over"


def p_abs(tol):
    """sum p |v| is at least tol / (2 * its largest factor); bounded by the cache's values instead."""
    return check.v_abs


CASES = [
    # lengths, new, page, heads, group, d
    ([1], [1], 16, 1, 1, 128),
    ([777], [1], 64, 2, 4, 128),
    ([300, 1, 0, 129, 128], [1, 1, 0, 1, 1], 16, 2, 2, 64),
    ([513, 40], [1, 1], 48, 1, 8, 96),
    ([200, 31], [5, 31], 32, 2, 1, 128),
    ([150, 260, 17], [17, 40, 3], 16, 2, 4, 64),
    ([90], [33], 16, 3, 5, 32),
    ([70, 70], [2, 2], 16, 2, 7, 80),
    ([45], [4], 16, 2, 1, 5),
    ([260], [100], 128, 1, 2, 100),
    ([1200], [3], 256, 1, 16, 128),
    ([64, 64, 64], [64, 64, 64], 16, 1, 1, 40),
]


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new,page,heads,group,d", CASES)
def test_attention(tq, codes, dtype, lengths, new, page, heads, group, d):
    import torch

    dt = dtype_of(dtype)
    c = Case(tq, lengths, new, page, heads, d, codes, seed=d)
    for t in (c.cache.k, c.cache.v):
        t.fill_(127)  # stale codes: NaN for e4m3
    for t in (c.cache.k_scale, c.cache.v_scale):
        t.fill_(float("nan"))
    c.fill(11)
    q = rand(12, c.rows, heads * group, d, dtype=dt, std=1.5)
    seen = torch.rand(c.rows, max(new), generator=torch.Generator().manual_seed(d)) < 0.6
    check.v_abs = float(torch.nan_to_num(c.cache.v_scale, 0.0).max()) * (127 if codes == "i8" else 448)
    for tree in (None, seen):
        ref, tol = reference(c, q, tree)
        got = c.cache.attention(q, c.batch, tree=None if tree is None else tq.tree_mask(tree).cuda())
        assert got.dtype == dt and got.shape == q.shape
        check(got, ref, tol, f"{lengths} {new} tree={tree is not None}")


def test_attention_of_many_ragged_sequences(tq):
    """More sequences than lanes, empty ones and rows behind the last among them; every share boundary
    falls somewhere."""
    import torch

    rng = np.random.default_rng(4)
    lengths = [int(x) for x in rng.integers(0, 400, 150)]
    new = [min(n, int(x)) for n, x in zip(lengths, rng.integers(0, 4, 150))]
    new[7] = lengths[7] = 0
    c = Case(tq, lengths, new, 16, 2, 64, "i8", ragged=True, extra=5)
    c.fill(21)
    q = rand(22, c.rows, 4, 64)
    out = torch.full_like(q, 3.0)
    c.cache.attention(q, c.batch, out=out)
    assert (out[-5:] == 3.0).all()
    ref, tol = reference(c, q)
    n = c.rows - 5
    check(out[:n], ref[:n], tol[:n])
    # one sequence at a time: the same rows, joined elsewhere
    for b in (0, 63, 64, 149):
        if not new[b]:
            continue
        one = tq.KVBatch(c.table[b:b + 1], c.batch.lengths[b:b + 1], new[b])
        rows = slice(int(c.offsets[b]), int(c.offsets[b + 1]))
        check(c.cache.attention(q[rows], one), ref[rows], tol[rows])


def test_attention_long(tq):
    """A long context: against 64 bits on the GPU, in f32 and bf16."""
    import torch

    length, heads, d = 70001, 2, 128
    c = Case(tq, [length], [1], 256, heads, d, "i8")
    c.fill(31)
    pos = torch.arange(length, device="cuda")
    pages = c.table[0, pos // 256].long()
    k = (c.cache.k[pages, :, pos % 256].double() * c.cache.k_scale[pages, :, pos % 256].double()[..., None]).transpose(0, 1).contiguous()
    v = (c.cache.v[pages, :, pos % 256].double() * c.cache.v_scale[pages, :, pos % 256].double()[..., None]).transpose(0, 1).contiguous()
    for dt in (torch.float32, torch.bfloat16):
        q = rand(32, 1, 8, d, dtype=dt, std=2.0)
        s = torch.matmul(q[0].double().view(heads, 4, d), k.transpose(1, 2).contiguous()) / math.sqrt(d)
        p = torch.softmax(s, -1)
        ref = torch.matmul(p, v).view(1, 8, d).cpu()
        size = torch.matmul(q[0].double().abs().view(heads, 4, d), k.abs().transpose(1, 2).contiguous()).max() / math.sqrt(d)
        pv = torch.matmul(p, v.abs()).view(1, 8, d).cpu()
        tol = 2 * 2.0 ** -24 * (float(size) * (d + 16) + 8 * (float(s.abs().max()) + 64)) * pv
        check.v_abs = pv
        check(c.cache.attention(q, c.batch), ref, tol)


@pytest.mark.parametrize("codes", ["i8", "fp8"])
def test_what_a_row_does_not_see_cannot_reach_it(tq, codes):
    """NaN and infinite keys and values among the new tokens reach the rows that see them and no others."""
    import torch

    new, d = 20, 64
    c = Case(tq, [50], [new], 16, 2, d, codes)
    b = c.all_tokens()
    k, v = rand(41, 50, 2, d), rand(42, 50, 2, d)
    q = rand(43, new, 4, d)
    seen = torch.ones(new, new, dtype=torch.bool)
    seen[::2, 7] = False
    seen[:, 11] = False
    seen[5, :] = False
    c.cache.write(k, v, b)
    clean = c.cache.attention(q, c.batch, tree=tq.tree_mask(seen).cuda())
    for bad, where in ((float("nan"), "v"), (float("inf"), "v"), (float("inf"), "k")):
        kk, vv = k.clone(), v.clone()
        for j in (7, 11):
            (kk if where == "k" else vv)[30 + j, :, 3] = bad
        c.cache.write(kk, vv, b)
        got = c.cache.attention(q, c.batch, tree=tq.tree_mask(seen).cuda())
        hit = seen[:, 7].cuda()
        assert torch.equal(got[~hit], clean[~hit])
        if codes == "fp8" and where == "v" and bad != bad:
            assert torch.isnan(got[hit][..., 3]).all() and torch.isfinite(got[hit][..., 4:]).all()
        elif bad == bad:
            assert torch.isnan(got[hit]).all()  # a scale of infinity: 0 * inf everywhere
    # value scales of 0 (no write leaves them) count as 1e-25: codes up to 448 of it
    c.cache.write(k, v, b)
    c.cache.v_scale.zero_()
    assert c.cache.attention(q, c.batch).abs().max() <= 448 * 1.01e-25


def test_attention_of_far_apart_scales(tq):
    """Values whose scales lie 2^40 apart, attended to the small ones: as exact as any."""
    import torch

    c = Case(tq, [96], [1], 32, 1, 64, "i8")
    b = c.all_tokens()
    k, v = rand(51, 96, 1, 64) * 0.1, rand(52, 96, 1, 64)
    v[::2] *= 2.0 ** 20
    v[1::2] *= 2.0 ** -20
    k[::2, :, 0] = -40.0
    k[1::2, :, 0] = 40.0
    c.cache.write(k, v, b)
    for factor in (1.0, 2.0 ** -60, 2.0 ** 60):
        q = torch.zeros(1, 2, 64, device="cuda")
        q[..., 0] = 40.0 * factor
        ref, tol = reference(c, q, scale=1.0 / (8 * factor))
        assert float(ref.abs().max()) < 1e-3
        check(c.cache.attention(q, c.batch, scale=1.0 / (8 * factor)), ref, tol)


def test_strides_streams_and_graphs(tq):
    """q read in place in a wider buffer; the whole step on another stream, and captured and replayed with
    new contents, gives what the eager calls give, bit for bit."""
    import torch

    h, hk, d, b = 8, 2, 128, 3
    lengths = [100, 257, 31]

    def step(c, buf, rot, batch):
        n = buf.shape[0]
        q, k, v = (x.view(n, -1, d) for x in (buf[:, :h * d], buf[:, h * d:(h + hk) * d], buf[:, (h + hk) * d:]))
        return c.cache.attention(c.cache.write_rotary(q, k, v, rot, batch), batch)

    def fresh():
        c = Case(tq, lengths, [1, 1, 1], 16, hk, d, "i8")
        c.fill(61)
        return c

    rot = tq.Rotary.from_base(d)
    bufs = [rand(70 + i, b, (h + 2 * hk) * d, dtype=torch.bfloat16) for i in range(4)]
    eager = fresh()
    want = [step(eager, x, rot, eager.batch).clone() for x in bufs]
    other = fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [step(other, x, rot, other.batch) for x in bufs]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    taped = fresh()
    buf = bufs[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step(taped, buf, rot, taped.batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(taped, buf, rot, taped.batch)
    taped.fill(61)
    for x, y in zip(bufs, want):
        buf.copy_(x)
        graph.replay()
        assert torch.equal(out, y)
        eager.fill(62)  # eager work between the replays
        torch.cuda.synchronize()


def test_a_decoded_sequence_is_the_prompt(tq):
    """Token by token, in chunks and at once: the same rows to f32 rounding, and the same cache, bit for bit."""
    import torch

    n, h, hk, d = 41, 4, 2, 64
    q, k, v = rand(81, n, h, d), rand(82, n, hk, d), rand(83, n, hk, d)
    rot = tq.Rotary.from_base(d)
    caches, outs = [], []
    for cuts in ([n], [1] * n, [16, 1, 20, 4]):
        c = Case(tq, [n], [n], 16, hk, d, "fp8")
        rows, at = [], 0
        for t in cuts:
            batch = tq.KVBatch(c.table, torch.tensor([at + t], dtype=torch.int32).cuda(), t)
            part = slice(at, at + t)
            rows.append(c.cache.attention(c.cache.write_rotary(q[part], k[part], v[part], rot, batch), batch))
            at += t
        caches.append(c)
        outs.append(torch.cat(rows))
    ref, tol = reference(caches[0], rot.apply(q, None, torch.arange(n, device="cuda"))[0])
    for c, o in zip(caches, outs):
        assert torch.equal(c.cache.k, caches[0].cache.k) and torch.equal(c.cache.v_scale, caches[0].cache.v_scale)
        check(o, ref, tol)


def test_no_tokens(tq):
    import torch

    c = Case(tq, [10], [1], 16, 2, 64, "i8")
    none = tq.KVBatch(c.table, c.batch.lengths, 0)
    x = torch.empty(0, 2, 64, device="cuda")
    c.cache.write(x, x, none)
    assert c.cache.attention(x, none).shape == (0, 2, 64)
    assert c.cache.read(none)[0].shape == (0, 2, 64)
    rot = tq.Rotary.from_base(64)
    assert rot.apply(x, x, torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)


# ------------------------------------------------------------------ many rows, and calls beside each other
@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,r,pairs,h,hk", [(128, 128, False, 4, 2), (80, 40, True, 3, 3), (64, 64, True, 2, 1), (33, 0, False, 1, 1)])
def test_many_rows_are_one_row_at_a_time(tq, codes, dtype, d, r, pairs, h, hk):
    """Ragged batches of some hundred rows, with rows that have no place and rows behind the last sequence: codes,
    turned q and what is read back are those of calls with one row, bit for bit."""
    import torch

    dt = dtype_of(dtype)
    lengths, new, extra, page = [150, 3, 70, 40, 12], [97, 3, 0, 40, 9], 6, 16
    a, b = (Case(tq, lengths, new, page, hk, d, codes, ragged=True, extra=extra) for _ in range(2))
    a.table[0, 4] = b.table[0, 4] = 10000  # positions 64..79 of the first sequence lie nowhere
    n = a.rows
    assert n >= 150
    q, k, v = rand(1, n, h, d, dtype=dt), rand(2, n, hk, d, dtype=dt), rand(3, n, hk, d, dtype=dt)
    rot = tq.Rotary.from_base(r, 500.0, pairs, scale=1.5)
    got = a.cache.write_rotary(q, k, v, rot, a.batch)
    row = 0
    for s, (length, t) in enumerate(zip(lengths, new)):
        for i in range(t):
            one = tq.KVBatch(b.table[s:s + 1], torch.tensor([length - t + i + 1], dtype=torch.int32).cuda(), 1)
            part = slice(row, row + 1)
            assert torch.equal(b.cache.write_rotary(q[part], k[part], v[part], rot, one), got[part]), row
            row += 1
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(a.cache, name), getattr(b.cache, name)), name
    out = tuple(torch.full((n, hk, d), 5.0, device="cuda", dtype=dt) for _ in range(2))
    a.cache.read(a.batch, dt, out)
    row = 0
    for s, (length, t) in enumerate(zip(lengths, new)):
        for i in range(t):
            one = tq.KVBatch(b.table[s:s + 1], torch.tensor([length - t + i + 1], dtype=torch.int32).cuda(), 1)
            for x, y in zip(out, b.cache.read(one, dt)):
                assert torch.equal(x[row:row + 1], y), row
                if 64 <= length - t + i < 80 and s == 0:
                    assert (y == 0).all()
            row += 1
    assert all((x[row:] == 5.0).all() for x in out)
    # a plain write leaves the same as a write that turns nothing
    c = Case(tq, lengths, new, page, hk, d, codes, ragged=True, extra=extra)
    e = Case(tq, lengths, new, page, hk, d, codes, ragged=True, extra=extra)
    c.cache.write(k, v, c.batch)
    e.cache.write_rotary(q, k, v, tq.Rotary.from_base(0), e.batch)
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(c.cache, name), getattr(e.cache, name)), name


def test_rotary_of_one_tensor_twice(tq):
    import torch

    x, pos = rand(1, 40, 3, 64), torch.arange(40, device="cuda") * 37
    rot = tq.Rotary.from_base(64)
    a, b = rot.apply(x, x, pos)
    assert torch.equal(a, b) and torch.equal(a, rot.apply(x, None, pos)[0]) and a.data_ptr() != b.data_ptr()


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new,page,heads,group,d", [
    ([1500], [100], 64, 1, 2, 128), ([700, 90], [70, 48], 32, 2, 1, 64), ([1000, 20, 400], [33, 20, 5], 16, 1, 2, 96),
    ([400], [129], 16, 1, 1, 33), ([600], [300], 48, 1, 1, 128), ([2000, 1], [9, 1], 16, 1, 5, 80)])
def test_attention_of_many_rows_and_keys(tq, codes, dtype, lengths, new, page, heads, group, d):
    """Tiles of 64 and 128 rows whose keys lie in several shares, behind each other and masked by trees of several
    words (one more than they need)."""
    import torch

    dt = dtype_of(dtype)
    c = Case(tq, lengths, new, page, heads, d, codes, seed=d)
    for t in (c.cache.k, c.cache.v):
        t.fill_(127)
    c.fill(13)
    q = rand(14, c.rows, heads * group, d, dtype=dt, std=1.5)
    seen = torch.rand(c.rows, (max(new) + 31) // 32 * 32 + 32, generator=torch.Generator().manual_seed(d)) < 0.3
    check.v_abs = float(c.cache.v_scale.max()) * (127 if codes == "i8" else 448)
    for tree in (None, seen):
        ref, tol = reference(c, q, tree)
        got = c.cache.attention(q, c.batch, tree=None if tree is None else tq.tree_mask(tree).cuda())
        check(got, ref, tol, f"{lengths} {new} tree={tree is not None}")


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("new,group", [(1, 4), (9, 3), (40, 1), (150, 1)])
def test_attention_skips_keys_without_a_page(tq, codes, new, group):
    """Keys on pages outside the cache are seen by nobody: the rest attended to alone, on other pages, gives the
    same up to the order of the sums."""
    import torch

    page, d, length = 16, 64, 500
    c = Case(tq, [length], [new], page, 2, d, codes)
    k, v = c.fill(17)
    lost = [0, 3, 4, 19]  # pages of the table, before the new tokens
    keep = [p for p in range(length) if p // page not in lost]
    e = Case(tq, [len(keep)], [new], page, 2, d, codes)
    e.cache.write(k[keep], v[keep], e.all_tokens())
    for i, p in enumerate(lost):
        c.table[0, p] = (-1, 1 << 30, c.cache.pages, -(1 << 31))[i]
    q = rand(18, new, 2 * group, d)
    ref, tol = reference(e, q)
    check(c.cache.attention(q, c.batch), ref, tol)
    check(e.cache.attention(q, e.batch), ref, tol)


def test_two_streams_and_two_graphs_beside_each_other(tq):
    """Calls on two streams at once, and two captured calls replayed by turns, each with the results of its own."""
    import torch

    jobs = []
    for i, (new, group, d) in enumerate([(1, 4, 128), (3, 2, 64), (60, 2, 128), (200, 1, 96)]):
        c = Case(tq, [900 + 7 * i, 300], [new, new], 32, 2, d, "i8")
        c.fill(90 + i)
        q = rand(95 + i, c.rows, 2 * group, d, dtype=torch.bfloat16)
        jobs.append((c, q, c.cache.attention(q, c.batch)))
    x, w = rand(99, 100, 512), tq.QuantizedLinear.from_tensors(rand(98, 300, 512), None, tq.QConfig.fp8_block())
    want = w(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for i, (c, q, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, c.cache.attention(q, c.batch), w(x)))
    torch.cuda.synchronize()
    for i, o, y in got:
        assert torch.equal(o, jobs[i][2]) and torch.equal(y, want)
    graphs, outs = [], []
    for c, q, _ in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((c.cache.attention(q, c.batch), w(x)))
        graphs.append(g)
    for order in ([0, 1, 2, 3], [3, 1, 2, 0], [2, 2, 0, 3, 1]):
        for o, y in outs:
            o.zero_()
            y.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for (o, y), (_, _, ref) in zip(outs, jobs):
            assert torch.equal(o, ref) and torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths,new,heads,group,d", [
    ([20000, 12345, 300], [40, 33, 40], 4, 1, 64), ([9000, 30000], [3, 1], 4, 4, 128), ([17000], [200], 8, 1, 128),
    ([4000] * 40 + [5], [1] * 41, 4, 2, 32)])
def test_attention_of_a_few_long_sequences(tq, dtype, lengths, new, heads, group, d):
    """Sequences of many more units than blocks, unequal ones: in units of several hundred keys, and (164 heads) in
    equal shares of the line; against 64 bits on the GPU, the bound of `reference`."""
    import torch

    dt = dtype_of(dtype)
    c = Case(tq, lengths, new, 64, heads, d, "i8", ragged=True)
    c.fill(33)
    q = rand(34, c.rows, heads * group, d, dtype=dt, std=1.5)
    got = c.cache.attention(q, c.batch)
    check.v_abs = float(c.cache.v_scale.max()) * 127
    for b, (length, t) in enumerate(zip(lengths, new)):
        pos = torch.arange(length, device="cuda")
        pages = c.table[b, pos // 64].long()
        k, v = ((x[pages, :, pos % 64, :d].double() * s[pages, :, pos % 64].double()[..., None]).transpose(0, 1).contiguous()
                for x, s in ((c.cache.k, c.cache.k_scale), (c.cache.v, c.cache.v_scale)))
        rows = slice(int(c.offsets[b]), int(c.offsets[b + 1]))
        qq = q[rows].double().view(t, heads, group, d).transpose(0, 1).reshape(heads, t * group, d)
        s = torch.matmul(qq, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        seen = pos[None] <= (length - t + torch.arange(t, device="cuda"))[:, None]
        s = s.masked_fill(~seen.repeat_interleave(group, 0)[None], -math.inf)
        size = (torch.matmul(qq.abs(), k.abs().transpose(1, 2).contiguous()) / math.sqrt(d)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        off = 2.0 ** -24 * ((d + 16) * size + 8 * (torch.where(s.isinf(), 0.0, s).abs().amax(-1, keepdim=True) + 64))
        ref, tol = (x.view(heads, t, group, d).transpose(0, 1).reshape(t, heads * group, d).cpu()
                    for x in (torch.matmul(p, v), 2 * off * torch.matmul(p, v.abs())))
        check(got[rows], ref, tol, f"sequence {b}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [3, 20, 50, 200])
def test_rows_of_far_apart_sizes(tq, dtype, new):
    """A row's result does not depend on how large the other rows of its tile are."""
    import torch

    dt = dtype_of(dtype)
    c = Case(tq, [300], [new], 16, 2, 64, "i8")
    c.fill(71)
    q = rand(72, new, 2, 64, dtype=dt)
    want = c.cache.attention(q, c.batch)
    far = q.clone()
    far[1::3] *= 2.0 ** 60
    far[2::3] *= 2.0 ** -60
    got = c.cache.attention(far, c.batch)
    assert torch.equal(got[::3], want[::3]) and torch.isfinite(got).all()


def test_what_a_descriptor_names_is_fixed(tq):
    """Replacing a tensor that the C calls were told of is refused (writing into it is not)."""
    import torch

    c = Case(tq, [10], [1], 16, 2, 64, "i8")
    rot = tq.Rotary.from_base(64)
    for x, name in ((c.cache, "k"), (c.cache, "v_scale"), (c.batch, "lengths"), (c.batch, "table"), (rot, "frequencies")):
        with pytest.raises(AttributeError):
            setattr(x, name, getattr(x, name) * 1)
    c.fill(1)
    q = rand(2, 1, 2, 64)
    a = c.cache.attention(q, c.batch)
    c.batch.lengths -= 3
    c.lengths = [7]
    ref, tol = reference(c, q)
    check(c.cache.attention(q, c.batch), ref, tol)
    assert not torch.equal(a, c.cache.attention(q, c.batch))


def test_batches_of_nothing(tq):
    """No sequences, a table without pages, and only rows behind the last sequence."""
    import torch

    c = Case(tq, [10], [1], 16, 2, 64, "i8")
    none = tq.KVBatch(torch.empty(0, 1, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 1,
                      torch.zeros(1, dtype=torch.int32, device="cuda"), 4)
    x, out = rand(1, 4, 2, 64), torch.full((4, 2, 64), 2.0, device="cuda")
    c.cache.write(x, x, none)
    c.cache.attention(x, none, out=out)
    c.cache.read(none, torch.float32, (out, out.clone()))
    assert (out == 2.0).all()
    empty = tq.KVBatch(torch.empty(2, 0, dtype=torch.int32, device="cuda"), torch.tensor([3, 0], dtype=torch.int32).cuda(), 2)
    c.cache.write(x, x, empty)
    assert (c.cache.attention(x, empty) == 0).all() and (c.cache.k == 0).all()
    assert all((t == 0).all() for t in c.cache.read(empty))


@pytest.mark.parametrize("codes", ["i8", "fp8"])
def test_a_cache_past_32_bits(tq, codes):
    """Pages whose rows and bytes lie past 2^31 and 2^32: what is written there is what is read and attended to, as
    on low pages."""
    import torch

    heads, d, page, pages = 16, 128, 64, 40000  # 5.2e9 bytes of keys, 41e6 rows
    big = tq.KVCache.allocate(pages, page, heads, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
    small = tq.KVCache.allocate(8, page, heads, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
    high = torch.tensor([[pages - 1, 20000, 33000, 16400]], dtype=torch.int32, device="cuda")
    low = torch.tensor([[5, 1, 7, 2]], dtype=torch.int32, device="cuda")
    n = 4 * page - 3
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    k, v = rand(1, n, heads, d), rand(2, n, heads, d)
    for cache, table in ((big, high), (small, low)):
        cache.write(k, v, tq.KVBatch(table, length, n))
    for new in (1, 9, 200):
        q = rand(3, new, heads, d)
        a, b = (cache.attention(q, tq.KVBatch(table, length, new)) for cache, table in ((big, high), (small, low)))
        assert torch.equal(a, b), new
        for x, y in zip(big.read(tq.KVBatch(high, length, new)), small.read(tq.KVBatch(low, length, new))):
            assert torch.equal(x, y) and float(x.abs().max()) > 1
    for i in range(4):
        assert torch.equal(big.k[int(high[0, i])], small.k[int(low[0, i])])


@pytest.mark.parametrize("longest,most", [(900, 1), (900, 4), (1300, 30), (500, 40)])
def test_attention_of_more_sequences_than_lanes(tq, longest, most):
    """Ragged batches of 130 sequences whose shares begin and end within them, or that are not cut."""
    import torch

    rng = np.random.default_rng(longest + most)
    lengths = [int(x) for x in rng.integers(0, longest + 1, 130)]
    lengths[3], lengths[100] = longest, 0
    new = [min(n, int(x)) for n, x in zip(lengths, rng.integers(0, most + 1, 130))]
    new[3], new[64] = min(most, longest), 0
    c = Case(tq, lengths, new, 16, 1, 64, "fp8", ragged=True, extra=3)
    c.fill(25)
    q = rand(26, c.rows, 2, 64)
    out = torch.full_like(q, 3.0)
    c.cache.attention(q, c.batch, out=out)
    assert (out[-3:] == 3.0).all()
    ref, tol = reference(c, q)
    check(out[:-3], ref[:-3], tol[:-3])
