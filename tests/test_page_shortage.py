"""Pools that run out of pages (tq_pages_grow_stored, tq_pages_lacking): tokens that found no page are nowhere for good, whatever
page a sequence gets later, and calls say what is missing."""
import random

import pytest

from test_cache_abi import refuse
from test_pages import Pool, at


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def test_refusals(abi):
    m, good = 1 << 20, Pool(1 << 20, 8, 16)
    for bad in (None, Pool(None, 8, 16), Pool(264, 8, 16), Pool(256, 0, 16), Pool(256, 8, 0)):
        refuse(abi, "tq_pages_grow_stored", at(bad), 2 * m, 4, 4, 3 * m, 4 * m, 2, None)
        refuse(abi, "tq_pages_lacking", at(bad), 2 * m, 4, 4, 3 * m, 2, 4 * m, None)
    for table, stride, width, batch in ((None, 4, 4, 2), (2 * m + 2, 4, 4, 2), (2 * m, 3, 4, 2), (2 * m, 4, -1, 2), (2 * m, 4, 4, -1)):
        refuse(abi, "tq_pages_grow_stored", at(good), table, stride, width, 3 * m, 4 * m, batch, None)
        refuse(abi, "tq_pages_lacking", at(good), table, stride, width, 3 * m, batch, 4 * m, None)
    refuse(abi, "tq_pages_grow_stored", at(good), 2 * m, 4, 4, 3 * m, 4 * m, 4097, None)
    for x in (None, 3 * m + 2):
        refuse(abi, "tq_pages_grow_stored", at(good), 2 * m, 4, 4, x, 4 * m, 2, None)
        refuse(abi, "tq_pages_grow_stored", at(good), 2 * m, 4, 4, 3 * m, x, 2, None)
        refuse(abi, "tq_pages_lacking", at(good), 2 * m, 4, 4, x, 2, 4 * m, None)
        refuse(abi, "tq_pages_lacking", at(good), 2 * m, 4, 4, 3 * m, 2, x, None)
    for first, size in ((2 * m, 4 * 8), (1 * m, 4 * 8)):  # over the table, over the holders
        for place in (first, first + size - 4, first - 4):
            refuse(abi, "tq_pages_grow_stored", at(good), 2 * m, 4, 4, 3 * m, place, 2, None)
            refuse(abi, "tq_pages_lacking", at(good), 2 * m, 4, 4, 3 * m, 2, place, None)
    refuse(abi, "tq_pages_lacking", at(good), 2 * m, 4, 4, 3 * m, 2, 3 * m + 4, None)
    abi.call("tq_pages_grow_stored", at(good), None, 0, 0, None, None, 3, None)
    abi.call("tq_pages_grow_stored", at(good), 2 * m, 4, 4, None, None, 0, None)
    abi.call("tq_pages_lacking", at(good), None, 0, 0, None, 0, None, None)


def ints(values):
    import torch

    return torch.tensor(values, dtype=torch.int32).cuda()


@pytest.mark.gpu
def test_a_copy_that_found_no_page_shows_nobody_elses_tokens(tq):
    """Fork without a page for the begun one, the parents end, the child grows: NaN lies wherever nothing was written."""
    import torch

    cache, pool = tq.KVCache.allocate(6, 16, 1, 32), tq.PagePool.allocate(6, 16)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(float("nan"))
    rows = lambda n: torch.randn(n, 1, 32, device="cuda")  # noqa: E731
    table, other = ints([[-1] * 5]), ints([[-1] * 5])
    pool.grow(table, ints([40]))
    pool.grow(other, ints([48]))
    cache.write(rows(40), rows(40), tq.KVBatch(table, ints([40]), 40))
    children, source, target = pool.fork(table, ints([40]), ints([0]))
    assert children.tolist() == [[0, 1, -1, -1, -1]] and target.tolist() == [-1]
    assert pool.lacking(children, ints([40])).tolist() == [1] and pool.lacking(children, ints([32])).tolist() == [0]
    cache.copy_pages(source, target)
    pool.free(table), pool.free(other)
    pool.grow(children, ints([60]), ints([40]))
    assert children.tolist() == [[0, 1, -1, 2, -1]]  # tokens 32 to 47 are nowhere, the next are on a page of their own
    assert pool.lacking(children, ints([60])).tolist() == [1] and pool.lacking(children, ints([81])).tolist() == [3]
    new = tq.KVBatch(children, ints([60]), 20)
    cache.write(rows(20), rows(20), new)
    for x in cache.read(tq.KVBatch(children, ints([60]), 60)):
        assert torch.isfinite(x).all() and (x[32:48] == 0).all() and (x[:32] != 0).any(2).all() and (x[48:] != 0).any(2).all()
    assert torch.isfinite(cache.attention(rows(20), new)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_every_place_holds_its_token_or_nothing(tq, seed):
    """Sequences that grow, fork and end in a pool that is always short: each token has a number of its own as its key and value,
    and what is read is that number, or 0 where it found no page."""
    import torch

    rng, page, width, pages = random.Random(seed), 16, 6, 6
    cache, pool = tq.KVCache.allocate(pages, page, 1, 32), tq.PagePool.allocate(pages, page)
    for t in (cache.k_scale, cache.v_scale):
        t.fill_(float("nan"))
    table, lives, count, lost = ints([[-1] * width for _ in range(3)]), [[], [], []], 0, 0

    def check():
        nonlocal lost
        n = [len(v) for v in lives]
        if not sum(n):
            return
        off = ints([sum(n[:i]) for i in range(len(n) + 1)])
        for x in cache.read(tq.KVBatch(table, ints(n), max(n), off, sum(n))):
            got, want = x[:, 0, 0].double(), torch.tensor([v or 0 for life in lives for v in life], dtype=torch.float64, device="cuda")
            assert ((got - want).abs() <= want * 2.0 ** -22).all()  # (the scale and the product, half a step each)
        lost += sum(v is None for life in lives for v in life)
        entries = table.tolist()
        assert pool.lacking(table, ints(n)).tolist() == [sum(e < 0 for e in row[:-(-v // page)]) for row, v in zip(entries, n)]
        held = [e for row in entries for e in row if e >= 0]
        assert pool.holders.tolist() == [held.count(e) for e in range(pages)]

    for step in range(25):
        had = [len(v) for v in lives]
        add = [rng.randint(0, min(20, page * width - v)) for v in had]
        pool.grow(table, ints([a + b for a, b in zip(had, add)]), ints(had))
        entries = table.tolist()
        for life, n, row in zip(lives, add, entries):
            for _ in range(n):
                count += 1
                life.append(count if row[len(life) // page] >= 0 else None)
        if sum(add):
            off = ints([sum(add[:i]) for i in range(4)])
            numbers = torch.tensor([life[i] or -1 for life, v in zip(lives, had) for i in range(v, len(life))], device="cuda", dtype=torch.float32)
            rows = numbers[:, None, None].expand(-1, 1, 32).contiguous()
            cache.write(rows, rows, tq.KVBatch(table, ints([len(v) for v in lives]), max(add), off, sum(add)))
        check()
        if step % 3 == 2:
            parents = [rng.randrange(3) for _ in range(3)]
            children, source, target = pool.fork(table, ints([len(v) for v in lives]), ints(parents))
            cache.copy_pages(source, target)
            entries = children.tolist()
            lives = [[v if entries[c][i // page] >= 0 else None for i, v in enumerate(lives[p])] for c, p in enumerate(parents)]
            pool.free(table)
            table = children
            check()
        gone = [rng.random() < 0.25 for _ in range(3)]
        pool.free(table, torch.tensor(gone).cuda())
        lives = [[] if x else v for v, x in zip(lives, gone)]
        check()
    assert lost  # (pages did run out under written tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,width,stride", [(1, 1, 1), (5, 130, 137), (4096, 3, 3)])
def test_what_is_lacking_and_what_stays_missing(tq, batch, width, stride):
    """Against lists: entries of stored tokens stay as they are, those behind are filled from behind the last page."""
    import torch

    rng, pages, page = random.Random(batch), 2000, 16
    rows = [[rng.choice([-1, -1, 5, pages, 1 << 30]) if rng.random() < 0.3 else rng.randrange(pages) for _ in range(width)] for _ in range(batch)]
    for row in rows:
        cut = rng.randrange(width + 1)
        row[cut:] = [-1] * (width - cut)
    lengths = [rng.choice([0, -3, rng.randint(1, page * width + 40)]) for _ in rows]
    stored = [rng.choice([0, -2, n, max(n, 0) // 2, n + 50]) for n in lengths]
    table = torch.full((batch, stride), -1, dtype=torch.int32).cuda()[:, :width]
    table.copy_(ints(rows))
    pool = tq.PagePool.allocate(pages, page)
    count = lambda n: max(-(-n // page), 0)  # noqa: E731
    missing = lambda: [sum(not 0 <= e < pages for e in row[:count(n)]) + max(count(n) - width, 0) for row, n in zip(rows, lengths)]  # noqa: E731
    assert pool.lacking(table, ints(lengths)).tolist() == missing()
    pool.grow(table, ints(lengths), ints(stored))
    free = iter(range(pages))
    for row, n, s in zip(rows, lengths, stored):
        need = min(count(n), width)
        have = max([i + 1 for i in range(need) if row[i] >= 0] + [min(count(s), need)])
        for i in range(have, need):
            row[i] = next(free, -1)
    assert table.tolist() == rows
    assert pool.lacking(table, ints(lengths)).tolist() == missing()


@pytest.mark.gpu
def test_captured_and_refused(tq):
    import torch

    pool, table = tq.PagePool.allocate(12, 16), ints([[-1] * 4] * 3)
    lengths, stored = ints([20, 0, 40]), ints([0, 0, 17])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pool.grow(table, lengths, stored), pool.lacking(table, lengths)
        pool.free(table)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.grow(table, lengths, stored)
        out = pool.lacking(table, lengths)
    for n, kept, want, missing in (([20, 0, 40], [0, 0, 17], [[0, 1, -1, -1], [-1] * 4, [-1, -1, 2, -1]], [0, 0, 2]),
                                   ([33, 64, 41], [20, 0, 40], [[0, 1, 3, -1], [4, 5, 6, 7], [-1, -1, 2, -1]], [0, 0, 2]),
                                   ([80, 64, 64], [33, 64, 41], [[0, 1, 3, 8], [4, 5, 6, 7], [-1, -1, 2, 9]], [1, 0, 2])):
        lengths.copy_(ints(n)), stored.copy_(ints(kept))
        graph.replay()
        torch.cuda.synchronize()
        assert table.tolist() == want and out.tolist() == missing
    for bad in (ints([1, 2]), lengths.long(), lengths.cpu(), None):
        with pytest.raises(tq.InvalidArgument):
            pool.lacking(table, bad)
        if bad is not None:
            with pytest.raises(tq.InvalidArgument):
                pool.grow(table, lengths, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", ["i8", "fp8"])
def test_kept_rows_that_found_no_page_end_the_sequence(tq, codes):
    """Drafts over a page that is missing, past the table or outside the cache: the rows of other branches that lie where such
    a row would go are not the sequence's.  A row that stays where it is nowhere leaves a gap that nobody sees."""
    import torch

    made = tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8
    # 30 tokens of which the last 20 are new: places 10 to 29, rows 0 to 5 on the first page, 6 to 19 on the second
    tables, paths, want = [], [], []
    for table, path, n in (([0, -1], [0, 2, 7], 2), ([1, -1], [0, 7, 9], 1), ([2, 99], [6, 7], 0), ([3, 4], [0, 7, 19], 3), ([-1, 5], [0, 7, 8], 3),
                           ([6, -1], [0, 1, 2, 3, 4, 5, 6, 7], 8), ([7, -1], [0, 1, 2, 3, 4, 6, 7], 5), ([-1, -1], [3, 9], 2), ([8, -1], [], 0)):
        tables.append(table), paths.append(path + [-1] * (8 - len(path))), want.append(10 + n)
    kept = ints([sum(r >= 0 for r in p) for p in paths])
    for heads, d in ((1, 32), (3, 128), (5, 80)):
        cache = tq.KVCache.allocate(10, 16, heads, d, made)
        new = tq.KVBatch(ints(tables), ints([30] * 9), 20)
        assert cache.keep(new, ints(paths), kept).tolist() == want, (heads, d)
    # 100 tokens, all new: the first lost row past a wave's first step, and past the table
    cache = tq.KVCache.allocate(10, 16, 2, 64, made)
    new = tq.KVBatch(ints([[0, 1, 2, 3, -1]] * 2), ints([100, 100]), 100)
    path = [list(range(1, 60)) + [70, 99], list(range(0, 80, 2)) + [-1] * 21]
    assert cache.keep(new, ints(path), ints([61, 40])).tolist() == [59, 32]
