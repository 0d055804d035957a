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


def test_what_adapters_write(abi):
    """out over the adapters' weights and scales and over the workspace (x, index and parts of y: see test_adapters)."""
    from test_adapters import desc

    m, count, parts, rank, k, n = 30, 4, 2, 32, 100, 60
    d = at(desc(a=40 * M, b=50 * M, scales=60 * M, count=count, parts=parts, rank=rank, k=k, n=n))
    need = abi.entry("tq_adapters_workspace_bytes")(d, m)
    assert need > 0
    for first, size in ((40 * M, 2 * count * parts * rank * 128), (50 * M, 2 * count * n * rank), (60 * M, 4 * count), (70 * M, need)):
        for out in both_ends(first, size, 4 * m * n):
            for y in (out, 4 * M):
                refuse(abi, "tq_adapters_add", d, 1 * M, 2, m, 2 * M, y, out, 70 * M, need, None)
                message(abi, (first, out))


def test_what_verification_writes(abi):
    """path, kept, next and the workspace over each other and over every input, rows of probabilities with their strides."""
    n, most, rows, vocab, stride = 3, 5, 11, 40000, 40008
    b = batch(abi, table=None, table_pages=0, lengths=256, offsets=1 * M, batch=n, max_tokens=most, tokens=rows)
    need = abi.entry("tq_verify_drafts_workspace_bytes")(at(b), vocab)
    reads = {"offsets": (1 * M, 4 * (n + 1)), "tokens": (2 * M, 8 * rows), "target": (10 * M, 4 * ((rows - 1) * stride + vocab)),
             "draft": (20 * M, 4 * ((rows - 1) * stride + vocab)), "parents": (3 * M, 4 * rows), "accept": (4 * M, 4 * rows), "final": (5 * M, 4 * n)}
    writes = {"workspace": (30 * M, need), "path": (6 * M, 4 * n * most), "kept": (7 * M, 4 * n), "next": (8 * M, 8 * n)}

    def no(draft, name, at_):
        w = {k: v[0] for k, v in writes.items()} | {name: at_}
        r = {k: v[0] for k, v in reads.items()} | ({} if draft else {"draft": None})
        refuse(abi, "tq_verify_drafts", at(b), r["tokens"], r["target"], stride, r["draft"], stride, 2, vocab, r["parents"], r["accept"],
               r["final"], w["workspace"], need, w["path"], w["kept"], w["next"], None)
        message(abi, (name, at_))

    for name, (_, length) in writes.items():
        step = {"workspace": 16, "next": 8}.get(name, 4)
        for other, (first, size) in (reads | writes).items():
            if other == name:
                continue
            for draft in (True, False):
                if not draft and other == "draft":
                    continue
                for place in (first, (first + size - 1) // step * step, (first - length) // step * step + step):
                    no(draft, name, place)


def test_what_a_pool_writes(abi):
    """Children, source and target over the table, lengths, parents, each other or the holders; the table over what calls read."""
    pages, n, children, width, stride = 40, 3, 5, 4, 9
    pool = at(Pool(1 * M, pages, 16))
    reads = {"table": (2 * M, 4 * ((n - 1) * stride + width)), "lengths": (3 * M, 4 * n), "parents": (4 * M, 4 * children), "holders": (1 * M, 4 * pages)}
    writes = {"out": (5 * M, 4 * children * width), "source": (6 * M, 4 * children), "target": (7 * M, 4 * children)}
    for name, (_, length) in writes.items():
        for other, (first, size) in (reads | writes).items():
            for place in both_ends(first, size, length) if other != name else ():
                w = {k: v[0] for k, v in writes.items()} | {name: place}
                refuse(abi, "tq_pages_fork", pool, 2 * M, stride, width, 3 * M, n, 4 * M, children, w["out"], w["source"], w["target"], None)
                message(abi, (name, place))
    for place in both_ends(*reads["holders"], reads["table"][1]):
        refuse(abi, "tq_pages_grow", pool, place, stride, width, 3 * M, n, None)
        message(abi, place)
        refuse(abi, "tq_pages_free", pool, place, stride, width, n, None, None)
        message(abi, place)
    for first, size in (reads["table"], reads["holders"]):
        for place in both_ends(first, size, 4 * n):
            refuse(abi, "tq_pages_grow", pool, 2 * M, stride, width, place, n, None)
            message(abi, place)
            refuse(abi, "tq_pages_free", pool, 2 * M, stride, width, n, max(place, first - n + 1), None)
            message(abi, place)


@pytest.mark.gpu
def test_neighbours_are_not_refused(tq):
    """Every input and output of a call one after the other in one buffer."""
    import torch

    abi, n, vocab, rows = tq._abi, 2, 50, 8
    sizes = {"tokens": 8 * rows, "next": 8 * n, "target": 4 * rows * vocab, "path": 4 * rows, "draft": 4 * rows * vocab, "kept": 4 * n, "accept": 4 * rows,
             "final": 4 * n, "parents": 4 * rows}
    buffer, where, first = torch.zeros(sum(sizes.values()), dtype=torch.uint8, device="cuda"), {}, 0
    for name, size in sizes.items():
        where[name], first = buffer[first:first + size], first + size
    as_ = lambda name, dtype: where[name].view(dtype)  # noqa: E731
    p = torch.softmax(torch.randn(rows, vocab, device="cuda"), 1)
    as_("target", torch.float32).copy_(p.flatten()), as_("draft", torch.float32).copy_(p.flatten().roll(1))
    as_("accept", torch.float32).fill_(0.5), as_("final", torch.float32).fill_(0.5)
    as_("parents", torch.int32).copy_(torch.tensor([-1, 0, 0, 1] * 2, dtype=torch.int32))
    as_("tokens", torch.int64).copy_(torch.arange(rows))
    new = tq.KVBatch(torch.zeros(n, 1, dtype=torch.int32).cuda(), torch.full((n,), 4, dtype=torch.int32).cuda(), 4)
    ptr = {k: v.data_ptr() for k, v in where.items()}
    abi.call("tq_verify_drafts", new._desc, ptr["tokens"], ptr["target"], vocab, ptr["draft"], vocab, 2, vocab, ptr["parents"], ptr["accept"],
             ptr["final"], None, 0, ptr["path"], ptr["kept"], ptr["next"], torch.cuda.current_stream().cuda_stream)
    want = tq.verify_drafts(torch.arange(rows, device="cuda"), p, new, torch.full((rows,), 0.5, device="cuda"), torch.full((n,), 0.5, device="cuda"),
                            p.flatten().roll(1).view(rows, vocab), as_("parents", torch.int32).clone())
    for name, w in zip(("path", "kept", "next"), want):
        assert torch.equal(as_(name, w.dtype).view(w.shape), w), name
    # keep's lengths between its paths and kept
    cache = tq.KVCache.allocate(2, 16, 1, 32)
    ints = torch.tensor([0, 2, 0, 3, -7, -7, 2, 2], dtype=torch.int32).cuda()
    new = tq.KVBatch(torch.tensor([[0], [1]], dtype=torch.int32).cuda(), torch.tensor([9, 9], dtype=torch.int32).cuda(), 4)
    abi.call("tq_kv_keep", cache._ref, new._desc, ints.data_ptr(), 2, 2, ints.data_ptr() + 24, ints.data_ptr() + 16,
             torch.cuda.current_stream().cuda_stream)
    assert ints.tolist() == [0, 2, 0, 3, 7, 7, 2, 2]
    # a pool's table behind its lengths, its holders behind both, and what a fork gives between parents and a strided table's rows
    ints = torch.zeros(64, dtype=torch.int32, device="cuda")
    ints[:2], ints[2:10], ints[12:24] = torch.tensor([17, 30]).cuda(), -1, 0
    pool, table, s = abi.page_pool_desc(ints[12:].data_ptr(), 12, 16), ints[2:10], torch.cuda.current_stream().cuda_stream
    abi.call("tq_pages_grow", pool, table.data_ptr(), 4, 4, ints.data_ptr(), 2, s)
    assert ints[:24].tolist() == [17, 30, 0, 1, -1, -1, 2, 3, -1, -1, 0, 0] + [1] * 4 + [0] * 8
    ints[24:26], ints[34:36] = torch.tensor([1, 0]).cuda(), 9
    at_ = lambda i: ints.data_ptr() + 4 * i  # noqa: E731
    abi.call("tq_pages_fork", pool, table.data_ptr(), 4, 4, ints.data_ptr(), 2, at_(24), 2, at_(26), at_(34), at_(36), s)
    assert ints[26:38].tolist() == [2, 4, -1, -1, 0, 5, -1, -1, 3, 1, 4, 5]
    abi.call("tq_pages_free", pool, at_(26), 4, 4, 2, None, s)
    assert ints[12:24].tolist() == [1] * 4 + [0] * 8 and ints[26:34].tolist() == [-1] * 8
