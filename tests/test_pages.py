"""Pages of the cache (tq_kv_keep, tq_kv_copy_pages, tq_pages_grow, tq_pages_fork, tq_pages_free): refusals on the CPU,
moves on the GPU against plain ones."""
import ctypes
import random

import pytest

from test_cache_abi import BAD_BATCH, BAD_CACHE, I64, PTR, batch, cache, refuse, structure

Pool = structure(("holders", PTR), ("pages", I64), ("page", I64))


HELD = []


def at(x):
    """The address of a structure, which stays."""
    HELD.append(x)
    return None if x is None else ctypes.addressof(x)


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def test_the_packed_descriptor_is_the_structure(abi):
    assert abi.page_pool_desc(1, 2, 3) == bytes(Pool(1, 2, 3))


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_caches(abi, kw):
    refuse(abi, "tq_kv_keep", at(cache(abi, **kw)), at(batch(abi)), 256, 1, 1, 256, 512, None)
    refuse(abi, "tq_kv_copy_pages", at(cache(abi, **kw)), 256, 256, 1, None)


@pytest.mark.parametrize("kw", BAD_BATCH)
def test_bad_batches(abi, kw):
    refuse(abi, "tq_kv_keep", at(cache(abi)), at(batch(abi, **kw)), 256, 1, 1, 256, 512, None)


def test_bad_moves(abi):
    c, b = cache(abi), batch(abi)
    for path, stride, width, kept, out in ((None, 1, 1, 256, 512), (256, 1, 1, None, 512), (258, 1, 1, 256, 512), (256, 1, 1, 258, 512),
                                           (256, 1, 1, 256, 514), (256, 0, 1, 256, 512), (256, 1, -1, 256, 512), (256, 1, 1 << 31, 256, 512),
                                           (256, 1, 1, 512, 256), (256, 1, 1, 512, 512)):  # (the batch's own lengths lie at 256)
        refuse(abi, "tq_kv_keep", at(c), at(b), path, stride, width, kept, out, None)
    abi.call("tq_kv_keep", at(c), at(batch(abi, batch=0, tokens=0)), None, 0, 0, None, None, None)
    many = batch(abi, batch=1 << 26, tokens=1 << 26)
    refuse(abi, "tq_kv_keep", at(c), at(many), 256, 1, 1, 256, 512, None)
    for source, target, n in ((None, 256, 1), (256, None, 1), (258, 256, 1), (256, 258, 1), (256, 256, -1), (256, 256, 1 << 40)):
        refuse(abi, "tq_kv_copy_pages", at(c), source, target, n, None)
    abi.call("tq_kv_copy_pages", at(c), None, None, 0, None)


def test_bad_pools(abi):
    good = Pool(256, 8, 16)
    for bad in (None, Pool(None, 8, 16), Pool(264, 8, 16), Pool(256, 0, 16), Pool(256, 1 << 31, 16), Pool(256, 8, 0), Pool(256, 8, 1 << 17)):
        refuse(abi, "tq_pages_grow", at(bad), 256, 4, 4, 256, 2, None)
        refuse(abi, "tq_pages_fork", at(bad), 256, 4, 4, 256, 2, 256, 2, 256, 256, 256, None)
        refuse(abi, "tq_pages_free", at(bad), 256, 4, 4, 2, None, None)
    for table, stride, width, batch_ in ((None, 4, 4, 2), (258, 4, 4, 2), (256, 3, 4, 2), (256, 4, -1, 2), (256, 4, 4, -1),
                                         (256, 1 << 31, 1 << 31, 2)):
        refuse(abi, "tq_pages_grow", at(good), table, stride, width, 256, batch_, None)
        refuse(abi, "tq_pages_fork", at(good), table, stride, width, 256, batch_, 256, 2, 256, 256, 256, None)
        refuse(abi, "tq_pages_free", at(good), table, stride, width, batch_, None, None)
    refuse(abi, "tq_pages_grow", at(good), 256, 4, 4, 256, 4097, None)
    refuse(abi, "tq_pages_grow", at(good), 256, 4, 4, None, 2, None)
    refuse(abi, "tq_pages_grow", at(good), 256, 4, 4, 258, 2, None)
    for i, v in ((5, None), (5, 258), (7, None), (7, 258), (8, 4097), (8, -1), (9, None), (9, 258), (10, None), (10, 258), (11, None), (11, 258)):
        args = [at(good), 256, 4, 4, 256, 2, 256, 2, 256, 256, 256, None]
        args[i - 1] = v
        refuse(abi, "tq_pages_fork", *args)
    abi.call("tq_pages_grow", at(good), None, 0, 0, None, 3, None)
    abi.call("tq_pages_free", at(good), None, 0, 4, 0, None, None)
    abi.call("tq_pages_fork", at(good), 256, 4, 4, 256, 2, None, 0, None, None, None, None)


# ------------------------------------------------------------------ what stays of drafts
def filled(tq, case, seed=0):
    """The case's cache with codes and scales that differ everywhere."""
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    for t in (case.cache.k, case.cache.v):
        t.copy_(torch.randint(0, 120, t.shape, generator=g, device="cuda").to(t.dtype))
    for t in (case.cache.k_scale, case.cache.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
    return {n: getattr(case.cache, n).clone() for n in ("k", "k_scale", "v", "v_scale")}


def moved(case, before, paths):
    """`before` with each sequence's rows of paths[b] at the first of its new places (None: as it is)."""
    table, want = case.table.tolist(), {n: t.clone() for n, t in before.items()}
    for b, path in enumerate(paths):
        for i, r in enumerate(path or []):
            src, dst = (case.lengths[b] - case.new[b] + x for x in (r, i))
            for n in want:
                want[n][table[b][dst // case.page], :, dst % case.page] = before[n][table[b][src // case.page], :, src % case.page]
    return want


def as_paths(paths, width):
    import torch

    rows = [(list(p) + [-1] * width)[:width] for p in paths]
    return torch.tensor(rows, dtype=torch.int32).view(len(paths), width).cuda(), torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("lengths,new,page,heads,d", [
    ([40], [8], 16, 2, 64), ([100, 33, 7], [30, 33, 1], 16, 3, 128), ([300, 20], [200, 20], 64, 1, 32), ([70, 70, 70, 70], [16] * 4, 48, 5, 80),
    ([5], [1], 16, 1, 1), ([90, 64], [70, 0], 32, 2, 100)])
def test_keep(tq, lengths, new, page, heads, d, codes):
    import torch
    from test_gpu_cache import Case

    rng = random.Random(d + heads)
    for trial in range(6):
        case = Case(tq, lengths, new, page, heads, d, codes, ragged=trial % 2 == 0 or 0 in new)
        before = filled(tq, case, trial)
        paths = []
        for n in new:
            k = rng.randint(0, n)
            paths.append(sorted(rng.sample(range(n), k)) if trial else list(range(n))[n // 2:])  # (the first: halves onto halves)
        path, kept = as_paths(paths, max(max(new), 1))
        got = case.cache.keep(case.batch, path, kept)
        want = moved(case, before, paths)
        for name, t in want.items():
            assert torch.equal(getattr(case.cache, name), t), (trial, name)
        assert got.tolist() == [v - n + len(p) for v, n, p in zip(lengths, new, paths)]


@pytest.mark.gpu
def test_paths_that_say_nothing_sound_leave_a_sequence_as_it_is(tq):
    import torch
    from test_gpu_cache import Case

    lengths, new = [50] * 9, [20] * 9
    case = Case(tq, lengths, new, 16, 2, 64, "i8")
    before = filled(tq, case)
    rows = torch.full((9, 20), -1, dtype=torch.int32)
    kept = [3, 3, 3, 3, -1, 21, 3, 20, 0]
    for i, p in enumerate([(0, 5, 5), (0, 7, 6), (0, 5, 20), (-1, 5, 6), (0, 5, 6), (0, 5, 6), (1, 5, 19), range(20), ()]):
        rows[i, :len(p)] = torch.tensor(list(p), dtype=torch.int32)
    got = case.cache.keep(case.batch, rows.cuda(), torch.tensor(kept, dtype=torch.int32).cuda())
    assert got.tolist() == [50] * 6 + [33, 50, 30]
    want = moved(case, before, [None] * 6 + [[1, 5, 19], range(20), []])
    for name, t in want.items():
        assert torch.equal(getattr(case.cache, name), t), name
    # more than 64 rows, the first mistake behind them; and kept past the paths' width
    case = Case(tq, [150] * 2, [150] * 2, 16, 1, 32, "fp8")
    before = filled(tq, case)
    path, kept = as_paths([list(range(1, 70)) + [69], list(range(1, 150))], 150)
    assert case.cache.keep(case.batch, path, kept).tolist() == [150, 149]
    want = moved(case, before, [None, range(1, 150)])
    assert torch.equal(case.cache.k, want["k"]) and torch.equal(case.cache.v_scale, want["v_scale"])
    path, _ = as_paths([range(100)] * 2, 100)
    assert case.cache.keep(case.batch, path, torch.tensor([101, 5], dtype=torch.int32).cuda()).tolist() == [150, 5]


@pytest.mark.gpu
def test_rows_without_a_place_do_not_move(tq):
    """Before position 0, past the table, on pages outside the cache, rows that do not fit; strided paths."""
    import torch
    from test_gpu_cache import Case

    case = Case(tq, [40, 40, 40], [30, 30, 30], 16, 2, 64, "i8")
    before = filled(tq, case)
    case.table[0, 1] = -3  # positions 16 to 31 of the first
    case.table[1, 2] = 999  # positions 32 to 39 of the second
    case.batch.lengths[2] = 20  # the first ten rows before position 0
    rows = torch.full((3, 40), 5, dtype=torch.int32).cuda()
    paths = [[2, 9, 25], [10, 22, 24], [4, 12, 20]]
    path, kept = as_paths(paths, 3)
    rows[:, 7:10] = path
    case.cache.keep(case.batch, rows[:, 7:10], kept)
    want = {n: t.clone() for n, t in before.items()}
    table = case.table.tolist()
    for b, p in enumerate(paths):
        for i, r in enumerate(p):
            src, dst = (int(case.batch.lengths[b]) - 30 + x for x in (r, i))
            ok = min(src, dst) >= 0 and all(0 <= table[b][x // 16] < case.cache.pages for x in (src, dst))
            if ok:
                for n in want:
                    want[n][table[b][dst // 16], :, dst % 16] = before[n][table[b][src // 16], :, src % 16]
    for n, t in want.items():
        assert torch.equal(getattr(case.cache, n), t), n


# ------------------------------------------------------------------ pages
@pytest.mark.gpu
@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("pages,page,heads,d,n", [(9, 16, 1, 1, 4), (40, 64, 8, 128, 17), (12, 48, 3, 100, 5), (6, 256, 2, 64, 1), (5, 16, 2, 32, 0)])
def test_copy_pages(tq, codes, pages, page, heads, d, n):
    import torch

    cache = tq.KVCache.allocate(pages, page, heads, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
    g = torch.Generator("cuda").manual_seed(d)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(0, 120, t.shape, generator=g, device="cuda").to(t.dtype))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
    order = random.Random(n).sample(range(pages), min(pages, 2 * n))
    source, target = order[:n], order[n:2 * n]
    target = (target + [-1] * n)[:n]
    if n > 3:  # pairs that are none, a page onto itself, one source for two
        source[0], target[1], source[2] = -1, pages, source[3]
    before = {k: getattr(cache, k).clone() for k in ("k", "k_scale", "v", "v_scale")}
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    cache.copy_pages(ints(source), ints(target))
    for name, t in before.items():
        want = t.clone()
        for s, e in zip(source, target):
            if 0 <= s < pages and 0 <= e < pages:
                want[e] = t[s]
        assert torch.equal(getattr(cache, name), want), name


class Model:
    """The pool as lists."""

    def __init__(self, pages, page):
        self.holders, self.page = [0] * pages, page

    def take(self):
        if 0 not in self.holders:
            return -1
        e = self.holders.index(0)
        self.holders[e] = 1
        return e

    def grow(self, table, lengths):
        for row, n in zip(table, lengths):
            have = max([i + 1 for i, e in enumerate(row) if e >= 0 and i < -(-n // self.page)], default=0)
            for i in range(have, min(-(-max(n, 0) // self.page), len(row))):
                row[i] = self.take()

    def fork(self, table, lengths, parents):
        children, source, target = [], [], []
        width = len(table[0])
        for p in parents:
            row = [-1] * width
            if 0 <= p < len(table):
                for i in range(min(max(lengths[p], 0) // self.page, width)):
                    row[i] = table[p][i]
                    if row[i] >= 0:
                        self.holders[row[i]] += 1
            children.append(row)
        for c, p in enumerate(parents):
            i = max(lengths[p], 0) // self.page if 0 <= p < len(table) else width
            begun = i < width and lengths[p] % self.page > 0 and table[p][i] >= 0
            e = self.take() if begun else -1
            source.append(table[p][i] if e >= 0 else -1)
            target.append(e)
            if e >= 0:
                children[c][i] = e
        return children, source, target

    def free(self, table, which):
        for row, gone in zip(table, which):
            for i, e in enumerate(row):
                if gone and e >= 0:
                    self.holders[e] = max(self.holders[e] - 1, 0)
                    row[i] = -1


@pytest.mark.gpu
@pytest.mark.parametrize("pages,page,width,batch", [(40, 16, 6, 3), (5000, 64, 70, 20), (17, 1, 9, 4), (40000, 16, 130, 300), (1, 16, 3, 2)])
def test_a_pool_through_forks_growth_and_ends(tq, pages, page, width, batch):
    import torch

    rng = random.Random(pages)
    pool, model = tq.PagePool.allocate(pages, page), Model(pages, page)
    for i in rng.sample(range(pages), pages // 3):  # pages of somebody else
        pool.holders[i] = model.holders[i] = 2
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    table, rows = torch.full((batch, width + 3), -1, dtype=torch.int32).cuda()[:, 1:width + 1], [[-1] * width for _ in range(batch)]
    lengths = [rng.choice([0, -5, 1, page, page + 1, rng.randint(1, page * width), page * width + 9]) for _ in range(batch)]
    for step in range(6):
        pool.grow(table, ints(lengths)), model.grow(rows, lengths)
        assert table.tolist() == rows and pool.holders.tolist() == model.holders, step
        parents = [rng.randrange(-1, batch + 1) for _ in range(rng.randint(1, 2 * batch))]
        got, want = pool.fork(table, ints(lengths), ints(parents)), model.fork(rows, lengths, parents)
        for a, b in zip(got, want):
            assert a.tolist() == b, step
        assert pool.holders.tolist() == model.holders, step
        pool.free(got[0]), model.free(want[0], [True] * len(parents))
        assert (got[0] == -1).all() and pool.holders.tolist() == model.holders, step
        gone = [rng.random() < 0.4 for _ in range(batch)]
        pool.free(table, torch.tensor(gone).cuda()), model.free(rows, gone)
        assert table.tolist() == rows and pool.holders.tolist() == model.holders, step
        lengths = [rng.randint(0, 2 * page) if x else min(n + rng.randint(0, 2 * page), width * page) for n, x in zip(lengths, gone)]
    pool.free(table), pool.free(table)  # twice: nothing more
    assert (pool.holders.cpu() >= 0).all() and sum(pool.holders.tolist()) == 2 * (pages // 3)


@pytest.mark.gpu
def test_as_many_sequences_as_a_call_takes_and_pages_that_run_out(tq):
    import torch

    n = 4096
    pool = tq.PagePool.allocate(3 * n // 2, 16)
    table = torch.full((n, 2), -1, dtype=torch.int32).cuda()
    lengths = torch.full((n,), 20, dtype=torch.int32).cuda()
    pool.grow(table, lengths)
    assert table.flatten()[:3 * n // 2].tolist() == list(range(3 * n // 2)) and (table.flatten()[3 * n // 2:] == -1).all()
    assert (pool.holders == 1).all()
    parents = torch.arange(n, dtype=torch.int32).cuda()
    children, source, target = pool.fork(table, lengths, parents)
    assert (source == -1).all() and (target == -1).all() and torch.equal(children[:, 0], table[:, 0]) and (children[:, 1] == -1).all()
    with pytest.raises(tq.InvalidArgument):
        pool.grow(torch.full((n + 1, 2), -1, dtype=torch.int32).cuda(), torch.zeros(n + 1, dtype=torch.int32).cuda())
    # pages that are not the pool's are not counted, nor freed; tables of no pages
    pool = tq.PagePool.allocate(4, 16)
    odd = torch.tensor([[7, 1 << 30, -1]], dtype=torch.int32).cuda()
    pool.grow(odd, torch.tensor([48], dtype=torch.int32).cuda())
    assert odd.tolist() == [[7, 1 << 30, 0]]
    pool.free(odd)
    assert odd.tolist() == [[-1] * 3] and pool.holders.tolist() == [0] * 4
    pool.grow(odd[:, :0], torch.tensor([48], dtype=torch.int32).cuda())
    assert pool.fork(odd[:, :0], torch.tensor([48], dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda())[0].shape == (2, 0)


@pytest.mark.gpu
def test_pools_that_python_refuses(tq):
    import torch

    holders = torch.zeros(9, dtype=torch.int32).cuda()
    for bad, page in ((holders[:0], 16), (holders, 0), (holders, -16), (holders, 65537), (holders[1:], 16), (holders.float(), 16)):
        with pytest.raises(tq.InvalidArgument):
            tq.PagePool(bad, page)


@pytest.mark.gpu
def test_a_pool_of_many_pages(tq):
    """The last pages of a million: found, and the lowest first."""
    import torch

    pages = (1 << 20) + 5
    pool = tq.PagePool.allocate(pages, 16)
    pool.holders.fill_(1)
    free = [0, 15, 16, 16383, 16384, 500000, pages - 5, pages - 1]
    pool.holders[free] = 0
    table = torch.full((3, 4), -1, dtype=torch.int32).cuda()
    pool.grow(table, torch.tensor([64, 1, 64], dtype=torch.int32).cuda())
    assert table.tolist() == [free[:4], [free[4], -1, -1, -1], free[5:] + [-1]]


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("most", [0.02, 0.0])  # of the numbers that accept: 0 accepts every first child
@pytest.mark.parametrize("codes", ["i8", "fp8"])
def test_drafts_from_positions_to_what_stays(tq, codes, most):
    """Prompts fork into samples, drafted trees are attended and verified, and what stays is what a cache that never
    saw the other branches holds, in every later token's attention too."""
    import torch
    from test_gpu_cache import rand

    page, heads, d, prompt, t, vocab = 16, 2, 64, 21, 6, 50
    made = tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8
    cache, plain = tq.KVCache.allocate(40, page, heads, d, made), tq.KVCache.allocate(40, page, heads, d, made)
    pool, ints = tq.PagePool.allocate(40, page), lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    rot = tq.Rotary.from_base(d, axes=tq.Rotary.axes_in_turn(d // 2, 3))
    x = rand(1, prompt, 3 * heads * d)
    part = lambda x, i: x[:, i * heads * d:(i + 1) * heads * d].view(-1, heads, d)  # noqa: E731
    pos = torch.stack([torch.arange(prompt).cuda(), torch.arange(prompt).cuda() // 5, torch.arange(prompt).cuda() % 5])
    table = torch.full((1, 4), -1, dtype=torch.int32).cuda()
    pool.grow(table, ints([prompt]))
    cache.write_rotary(part(x, 0), part(x, 1), part(x, 2), rot, tq.KVBatch(table, ints([prompt]), prompt), pos)
    samples, source, target = pool.fork(table, ints([prompt]), ints([0, 0, 0]))
    cache.copy_pages(source, target)
    pool.free(table)
    lengths = ints([prompt + t] * 3)
    pool.grow(samples, lengths)
    y = rand(2, 3 * t, 3 * heads * d)
    parents = [-1, 0, 0, 1, 2, 3]
    depth = [0, 1, 1, 2, 2, 3]
    at_ = torch.tensor([prompt + v for v in depth] * 3).cuda().expand(3, 3 * t)
    new = tq.KVBatch(samples, lengths, t)
    q = cache.write_rotary(part(y, 0), part(y, 1), part(y, 2), rot, new, at_)
    seen = torch.zeros(t, t, dtype=torch.bool)
    for i, p in enumerate(parents):
        seen[i] = seen[p] if p >= 0 else False
        seen[i, i] = True
    tree_out = cache.attention(q, new, tree=tq.tree_mask(seen.repeat(3, 1).cuda()))
    g = torch.Generator("cuda").manual_seed(7)
    target_p = torch.softmax(torch.randn(3 * t, vocab, generator=g, device="cuda"), 1)
    tokens = torch.randint(0, vocab, (3 * t,), generator=g, device="cuda")
    accept = torch.rand(3 * t, generator=g, device="cuda") * most
    path, kept, token = tq.verify_drafts(tokens, target_p, new, accept, torch.rand(3, generator=g, device="cuda"), None, ints(parents * 3))
    lengths = cache.keep(new, path, kept)
    assert most or (kept == 4).all()  # rows 0, 1, 3, 5
    pool.grow(samples, lengths + 1)
    z = rand(3, 3, 3 * heads * d)
    nxt = tq.KVBatch(samples, lengths + 1, 1)
    after = (lengths.long()[None]).expand(3, 3)
    out = cache.attention(cache.write_rotary(part(z, 0), part(z, 1), part(z, 2), rot, nxt, after), nxt)
    for b in range(3):  # the same tokens one after the other in a cache of their own
        rows = path[b, :int(kept[b])].tolist()
        own = torch.arange(b * 4, b * 4 + 4, dtype=torch.int32).cuda().view(1, 4)
        plain.write_rotary(part(x, 0), part(x, 1), part(x, 2), rot, tq.KVBatch(own, ints([prompt]), prompt), pos)
        for i, r in enumerate(rows):
            one, place = y[b * t + r:b * t + r + 1], tq.KVBatch(own, ints([prompt + i + 1]), 1)
            o = plain.attention(plain.write_rotary(part(one, 0), part(one, 1), part(one, 2), rot, place, at_[:, b * t + r:b * t + r + 1]), place)
            # the same keys, another split of the sums: 2^-20 of the values
            assert (o - tree_out[b * t + r]).abs().max() <= 2.0 ** -20 * 8 * float(part(y, 2).abs().max())
        last = tq.KVBatch(own, ints([prompt + len(rows) + 1]), 1)
        one = z[b:b + 1]
        o = plain.attention(plain.write_rotary(part(one, 0), part(one, 1), part(one, 2), rot, last, after[:, b:b + 1]), last)
        assert (o - out[b]).abs().max() <= 2.0 ** -20 * 8 * float(part(y, 2).abs().max())
        everything = tq.KVBatch(own, last.lengths, prompt + len(rows) + 1)
        mine = tq.KVBatch(samples[b:b + 1], last.lengths, prompt + len(rows) + 1)
        for a, c in zip(cache.read(mine), plain.read(everything)):
            assert torch.equal(a, c)
    pool.free(samples)
    assert (pool.holders == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", ["i8", "fp8"])
def test_caches_past_32_bit_offsets(tq, codes):
    """5 GB of codes: pages and rows on both sides of 2^31 and 2^32 bytes."""
    import torch

    pages, page, heads, d = 80000, 64, 8, 128
    cache = tq.KVCache.allocate(pages, page, heads, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
    some = [0, 32767, 32768, 65535, 65536, pages - 1, pages - 2, 5]
    g = torch.Generator("cuda").manual_seed(1)
    for t in (cache.k, cache.v):
        t[some] = torch.randint(0, 100, (len(some), heads, page, d), generator=g, device="cuda").to(t.dtype)
    for t in (cache.k_scale, cache.v_scale):
        t[some] = torch.rand(len(some), heads, page, generator=g, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    names = ("k", "k_scale", "v", "v_scale")
    cache.copy_pages(ints([65536, 32768, pages - 1]), ints([40000, 70000, 1]))
    for n in names:
        t = getattr(cache, n)
        assert torch.equal(t[40000], t[65536]) and torch.equal(t[70000], t[32768]) and torch.equal(t[1], t[pages - 1]), n
    before = {n: getattr(cache, n).clone()[[pages - 2, 32767]] for n in names}
    new = tq.KVBatch(ints([[pages - 2, 32767]]), ints([120]), 100)  # positions 20 to 119
    assert cache.keep(new, ints([[3, 50, 99]]), ints([3])).tolist() == [23]
    for n in names:
        t = getattr(cache, n)
        for i, r in enumerate((3, 50, 99)):
            src = 20 + r
            assert torch.equal(t[pages - 2][:, 20 + i], before[n][src // page][:, src % page]), (n, i)


@pytest.mark.gpu
def test_keeping_and_pages_captured_and_replayed(tq):
    """A step's keep, growth, fork, copy and end in a graph: each replay as the eager calls on the same state."""
    import torch
    from test_gpu_cache import Case

    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731

    def state():
        case = Case(tq, [40, 33], [12, 12], 16, 2, 64, "i8", spare=20)
        filled(tq, case, 3)
        pool = tq.PagePool.allocate(case.cache.pages, 16)
        pool.holders[case.table.flatten().long()] = 1
        table = torch.cat([case.table, torch.full((2, 3), -1, dtype=torch.int32, device="cuda")], 1)
        return case, pool, table, ints([[0, 2, 5, 9], [0, 1, 7, -1]]), ints([4, 3]), ints([1, 0, 1])

    def step(case, pool, table, path, kept, parents):
        lengths = case.cache.keep(case.batch, path, kept)
        pool.grow(table, lengths + 20)
        children, source, target = pool.fork(table, lengths, parents)
        case.cache.copy_pages(source, target)
        had = children.clone()
        pool.free(children)
        return lengths, had, source, target

    eager, still = state(), state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*state())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*still)
    for i in range(4):
        for x in (eager, still):
            x[0].batch.lengths.copy_(ints([40 + 3 * i, 33 + i]))
        want = step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        assert torch.equal(eager[1].holders, still[1].holders) and torch.equal(eager[2], still[2])
        for n in ("k", "k_scale", "v", "v_scale"):
            assert torch.equal(getattr(eager[0].cache, n), getattr(still[0].cache, n)), (i, n)
