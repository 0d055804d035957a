"""Verification of drafted tokens (tq_verify_drafts): refusals on the CPU, decisions on the GPU against a walk in 64 bits."""
import ctypes
import math

import pytest

from test_cache_abi import batch, refuse


HELD = []
SMALL = 32768  # the largest vocabulary of one launch


def at(x):
    """The address of a structure, which stays."""
    HELD.append(x)
    return None if x is None else ctypes.addressof(x)


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def test_refusals(abi):
    b = batch(abi)
    good = [at(b), 256, 256, 100000, 256, 100000, 2, 100000, 256, 256, 256, 256, 1 << 20, 256, 256, 256, None]

    def no(**kw):
        args = list(good)
        for i, v in kw.items():
            args[int(i[1:])] = v
        refuse(abi, "tq_verify_drafts", *args)

    no(_0=None)
    for kw in (dict(batch=-1), dict(tokens=-1), dict(max_tokens=-1), dict(tokens=5), dict(offsets=258, tokens=5), dict(batch=1 << 31, tokens=1 << 31)):
        bad = batch(abi, **kw)
        no(_0=at(bad))
        assert abi.entry("tq_verify_drafts_workspace_bytes")(at(bad), 100) == -1
    for i, v in ((1, None), (1, 260), (2, None), (2, 258), (3, -1), (4, 258), (5, -1), (6, 3), (6, 7), (7, 0), (7, -5), (7, 1 << 31), (8, 258),
                 (9, None), (9, 258), (10, None), (10, 258), (11, None), (11, 264), (12, 8), (13, None), (13, 258), (14, None), (14, 258),
                 (15, None), (15, 260)):
        no(**{f"_{i}": v})
    assert abi.entry("tq_verify_drafts_workspace_bytes")(at(b), 100000) % 16 == 0
    assert abi.entry("tq_verify_drafts_workspace_bytes")(at(b), SMALL) == 0 < abi.entry("tq_verify_drafts_workspace_bytes")(at(b), SMALL + 1)
    no(_7=SMALL, _2=None), no(_7=SMALL, _13=None)
    huge = batch(abi, batch=1 << 22, max_tokens=1, tokens=1 << 22)  # more blocks than a launch has
    no(_0=at(huge), _12=1 << 62)
    wide = batch(abi, batch=1 << 20, max_tokens=1, tokens=1 << 20)
    no(_0=at(wide), _7=1 << 30, _12=1 << 62)
    none = batch(abi, batch=0, tokens=0)
    abi.call("tq_verify_drafts", at(none), *([None] * 2), 0, None, 0, 2, 100, *([None] * 4), 0, None, None, None, None)


def walk(tokens, p, q, parents, accept, final):
    """One sequence by the definition: lists, p and q lists of rows of Python floats (64 bits)."""
    if not tokens:
        return [], -1
    node, path, tried = 0, [0], []
    pos = lambda v: v if v > 0 else 0.0  # noqa: E731  (NaN: 0)
    p, q = [[pos(v) for v in row] for row in p], None if q is None else [[pos(v) for v in row] for row in q]
    a, w = 0.0, 1.0
    for t in range(1, len(tokens)):
        if parents[t] != node:
            continue
        x = tokens[t]
        inside = 0 <= x < len(p[node])
        if q is None:
            px = p[node][x] if inside and x not in tried else 0.0
            yes = accept[t] * w < px
        else:
            px, qx = (p[node][x], q[node][x]) if inside else (0.0, 0.0)
            yes = accept[t] * qx * w < px - a * qx
        if yes:
            node, a, w, tried = t, 0.0, 1.0, []
            path.append(t)
        elif q is None:
            w -= px
            tried.append(x)
        else:
            a += w
            w = math.fsum(pos(v - a * u) for v, u in zip(p[node], q[node]))
    left = [0.0 if i in tried else pos(v) for i, v in enumerate(p[node])] if q is None else \
        [pos(v - a * u) for v, u in zip(p[node], q[node])]
    if not math.fsum(left) > 0:
        left = [pos(v) for v in p[node]]
    total, run = math.fsum(left), 0.0
    if not total > 0:
        return path, -1
    for i, v in enumerate(left):
        run += v
        if v > 0 and run > final * total:
            return path, i
    return path, max(i for i, v in enumerate(left) if v > 0)


def make(counts, vocab, tree, draft, dtype, seed, width=3, std=2.0):
    """Tokens that are often accepted: drawn from the draft's probabilities, or its likeliest."""
    import torch

    g = torch.Generator().manual_seed(seed)
    rows = sum(counts)
    z = torch.randn(max(rows, 1), vocab, generator=g) * std
    p = torch.softmax(z, 1).to(dtype)
    q = torch.softmax(z + torch.randn(z.shape, generator=g) * 0.7, 1).to(dtype)
    parents, tokens, first = [], [], 0
    for n in counts:
        for t in range(n):
            up = t - 1 if not tree or t == 0 else int(torch.randint(max(0, t - 2 * width), t, (1,), generator=g))
            parents.append(up)
            row = q[first + max(up, 0)].float()
            tokens.append(int(torch.multinomial(row, 1, generator=g)) if draft else
                          int(row.topk(min(width, vocab)).indices[int(torch.randint(0, min(width, vocab), (1,), generator=g))]))
        first += n
    return (torch.tensor(tokens, dtype=torch.int64), p[:rows], q[:rows] if draft else None, torch.tensor(parents, dtype=torch.int32),
            torch.rand(rows, generator=g), torch.rand(len(counts), generator=g))


def batch_of(tq, counts, most=None, ragged=True, extra=0):
    import torch

    b, most = len(counts), max(counts) if most is None else most
    table, lengths = torch.zeros(b, 1, dtype=torch.int32).cuda(), torch.tensor(counts, dtype=torch.int32).cuda()
    if not ragged:
        return tq.KVBatch(table, lengths, most)
    off = torch.tensor([sum(counts[:i]) for i in range(b + 1)], dtype=torch.int32).cuda()
    return tq.KVBatch(table, lengths, most, off, sum(counts) + extra)


def check(tq, counts, tokens, p, q, parents, accept, final, chain, new=None):
    import torch

    new = new or batch_of(tq, counts)
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    call = lambda p, q: tq.verify_drafts(cuda(tokens), p, new, cuda(accept), cuda(final), q, None if chain else cuda(parents))  # noqa: E731
    path, kept, token = call(cuda(p), cuda(q))
    assert path.dtype == kept.dtype == torch.int32 and token.dtype == torch.int64
    if p.shape[1] <= SMALL:  # tokens that never come change nothing, and take the form of large vocabularies
        wider = lambda x: None if x is None else torch.nn.functional.pad(x.cuda(), (0, SMALL + 9 - x.shape[1]))  # noqa: E731
        for a, b in zip((path, kept, token), call(wider(p), wider(q))):
            assert torch.equal(a, b)
    path, kept, token, first, longest = path.tolist(), kept.tolist(), token.tolist(), 0, 0
    rows = lambda x, a, n: None if x is None else x[a:a + n].double().tolist()  # noqa: E731
    for i, n in enumerate(counts):
        part = slice(first, first + n)
        want, following = walk(tokens[part].tolist(), rows(p, first, n), rows(q, first, n), parents[part].tolist(),
                               accept[part].double().tolist(), float(final[i]))
        assert kept[i] == len(want) and path[i] == want + [-1] * (new.tokens - len(want)), (i, path[i], want)
        assert token[i] == following, i
        first, longest = first + n, max(longest, len(want))
    return longest


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("counts,vocab", [([1], 7), ([6], 1000), ([5, 1, 8, 3], 1025), ([2], 1), ([3, 0, 4], 33), ([9] * 5, 4100),
                                          ([64, 65, 70], 40), ([150, 1, 40], 12), ([4, 7], 20004), ([6, 2, 9], 32768), ([5, 8], 32769)])
def test_decisions(tq, counts, vocab, tree, draft, dtype):
    import torch

    for seed in range(3):
        check(tq, counts, *make(counts, vocab, tree, draft, getattr(torch, dtype), 100 * seed + vocab), not tree)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_deep_trees_and_chains_are_followed(tq, draft):
    """Numbers near 0 accept whatever has mass: paths of many rows, over 64 rows too."""
    import torch

    counts = [200, 64, 129]
    tokens, p, q, parents, accept, final = make(counts, 6, False, draft, torch.float32, 3, std=0.3)
    assert check(tq, counts, tokens, p, q, parents, accept * 1e-3, final, True) > 64
    assert check(tq, counts, tokens, p, q, parents, accept * 1e-3, final, False) > 64  # the same as a tree
    tokens, p, q, parents, accept, final = make(counts, 6, True, draft, torch.float32, 4, width=2, std=0.3)
    check(tq, counts, tokens, p, q, parents, accept * 0.2, final, False)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_siblings_that_are_all_turned_down_and_tokens_of_no_vocabulary(tq, draft):
    """One root with 100 children: what is left shrinks child by child; repeated tokens, tokens outside, bad parents."""
    import torch

    n, vocab = 101, 300
    tokens, p, q, parents, accept, final = make([n], vocab, True, draft, torch.float32, 9)
    parents[1:] = 0
    tokens[3], tokens[5], tokens[7], tokens[70], tokens[71] = tokens[2], -1, vocab, tokens[2], 1 << 40
    parents[10], parents[11], parents[12] = 10, 50, -7
    for top in (1.0, 0.0):  # 1: never accepted while what is left is more than the child's own
        u = torch.full((n,), top) if top else accept * 0.05
        check(tq, [n], tokens, p, q, parents, u, final, False)


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [False, True])
def test_probabilities_that_are_none(tq, tree):
    """Rows of zeros, NaN, negative numbers, q above p everywhere (nothing left), u and final of 0."""
    import torch

    for draft in (False, True):
        for kind in range(6):
            counts = [4, 4, 1]
            tokens, p, q, parents, accept, final = make(counts, 50, tree, draft, torch.float32, 30 + kind)
            if kind == 0:
                p.zero_()
            elif kind == 1:
                p[:, ::3] = float("nan")
            elif kind == 2:
                p[:, ::2] *= -1
            elif kind == 3:
                accept.fill_(1.0)
                if draft:
                    q.copy_(p)
            elif kind == 4:
                accept.zero_(), final.zero_()
                p[:, :7] = 0
            else:
                final.fill_(1.0 - 2.0 ** -24)
            check(tq, counts, tokens, p, q, parents, accept, final, not tree)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("tree,draft", [(False, True), (True, False), (True, True)])
def test_single_probabilities_that_are_none_count_as_zeros(tq, tree, draft, dtype):
    """Of the drafted tokens themselves and of others, in the target and in the draft: as if zeros stood there (the numbers
    that accept are small: a child whose draft probability is none is accepted where the target's is above 0)."""
    import torch

    for seed, none in enumerate((float("nan"), -0.25, -float("inf"))):
        counts = [12, 9, 16]
        tokens, p, q, parents, accept, final = make(counts, 300, tree, draft, getattr(torch, dtype), 60 + seed, width=5)
        accept *= 0.3
        first = torch.tensor(sum(([sum(counts[:i])] * n for i, n in enumerate(counts)), []))
        at_parent = first + parents.clamp(min=0)
        p[at_parent[::3], tokens[::3]] = none
        p[:, 7::11] = none
        if draft:
            q[at_parent[::2], tokens[::2]] = none
            q[:, 5::9] = none
        check(tq, counts, tokens, p, q, parents, accept, final, not tree)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [2000, 34000])
def test_infinite_probabilities_end(tq, vocab):
    """What they give is unspecified, a token of the vocabulary or -1."""
    import torch

    tokens, p, q, parents, accept, final = (None if x is None else x.cuda() for x in make([5, 5], vocab, False, True, torch.float32, 5))
    p[:, 77] = float("inf")
    for draft in (None, q):
        path, kept, token = tq.verify_drafts(tokens, p, batch_of(tq, [5, 5]), accept, final, draft)
        assert (token >= -1).all() and (token < vocab).all() and (kept >= 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [64, 33000])
def test_rows_that_do_not_fit_and_rows_behind(tq, draft, vocab):
    """Offsets that run out of the call or past max_tokens: kept 0, token -1; the other sequences as ever."""
    import torch

    counts = [5, 5, 5]
    tokens, p, q, parents, accept, final = make(counts, vocab, True, draft, torch.float32, 6)
    cuda = [None if x is None else x.cuda() for x in (tokens, p, q, parents, accept, final)]
    want = tq.verify_drafts(cuda[0], cuda[1], batch_of(tq, counts), cuda[4], cuda[5], cuda[2], cuda[3])
    table, lengths = torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    for off, most, fits in (([0, 5, 10, 16], 5, [1, 1, 0]), ([-1, 5, 10, 15], 9, [0, 1, 1]), ([0, 5, 10, 15], 4, [0, 0, 0]),
                            ([0, 5, 4, 15], 5, [1, 0, 0]), ([2**31 - 1, 5, 10, 15], 5, [0, 1, 1])):
        new = tq.KVBatch(table, lengths, most, torch.tensor(off, dtype=torch.int32).cuda(), 15)
        path, kept, token = tq.verify_drafts(cuda[0], cuda[1], new, cuda[4], cuda[5], cuda[2], cuda[3])
        for i, ok in enumerate(fits):
            if ok:
                assert kept[i] == want[1][i] and token[i] == want[2][i] and torch.equal(path[i, :4], want[0][i, :4])
            else:
                assert kept[i] == 0 and token[i] == -1 and (path[i] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [1024, 40000])
def test_strides_and_other_streams(tq, dtype, vocab):
    import torch

    counts = [6, 4]
    tokens, p, q, parents, accept, final = make(counts, vocab, True, True, getattr(torch, dtype), 8)
    args = [x.cuda() for x in (tokens, p, q, parents, accept, final)]
    new = batch_of(tq, counts)
    want = tq.verify_drafts(args[0], args[1], new, args[4], args[5], args[2], args[3])
    for skip, wide in ((1, vocab + 3), (0, vocab + 7), (4, 2 * vocab)):
        big = [torch.zeros(10 * wide + skip, dtype=p.dtype, device="cuda") for _ in range(2)]
        view = [b[skip:].view(10, wide)[:, :vocab] for b in big]
        view[0].copy_(args[1]), view[1].copy_(args[2])
        for a, b in zip(want, tq.verify_drafts(args[0], view[0], new, args[4], args[5], view[1], args[3])):
            assert torch.equal(a, b)
    turned = [x.t().contiguous().t() for x in args[1:3]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tq.verify_drafts(args[0], turned[0], new, args[4], args[5], turned[1], args[3])
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("tree,draft", [(False, True), (True, False), (True, True)])
def test_what_comes_out_is_the_targets_distribution(tq, tree, draft):
    """The token after the root (an accepted child's, or the one drawn) is distributed as the target says, whatever
    the draft: 60000 sequences; counts are binomial, 5 standard deviations for each of 4 tokens (2e-6 in all)."""
    import torch

    n, b, vocab = 4, 60000, 4
    g = torch.Generator("cuda").manual_seed(4)
    p = torch.tensor([0.5, 0.25, 0.2, 0.05], device="cuda").expand(n * b, vocab)
    q = torch.tensor([0.1, 0.2, 0.3, 0.4], device="cuda").expand(n * b, vocab)
    tokens = torch.multinomial(q[0], n * b, replacement=True, generator=g)
    parents = torch.tensor([-1, 0, 0, 0] if tree else [-1, 0, 1, 2], dtype=torch.int32).repeat(b).cuda()
    accept, final = torch.rand(n * b, device="cuda", generator=g), torch.rand(b, device="cuda", generator=g)
    new = tq.KVBatch(torch.zeros(b, 1, dtype=torch.int32).cuda(), torch.full((b,), n, dtype=torch.int32).cuda(), n)
    if not draft:
        tokens = tokens.view(b, n)
        tokens[:, 1:] = torch.tensor([3, 1, 0]).cuda()  # whatever is tried first
        tokens = tokens.reshape(-1)
    path, kept, token = tq.verify_drafts(tokens, p, new, accept, final, q if draft else None, parents if tree else None)
    second = torch.where(kept > 1, tokens.view(b, n).gather(1, path[:, 1:2].clamp_min(0).long())[:, 0], token)
    for i in range(vocab):
        want = b * float(p[0, i])
        assert abs(int((second == i).sum()) - want) < 5 * math.sqrt(want * (1 - float(p[0, i])))


@pytest.mark.gpu
@pytest.mark.parametrize("tree,draft", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("vocab", [3001, 33000])
def test_captured_and_replayed(tq, tree, draft, vocab):
    import torch

    counts = [7, 3, 5]
    sets = [make(counts, vocab, tree, draft, torch.float32, s) for s in range(4)]
    new, still = batch_of(tq, counts), [None if x is None else x.cuda() for x in sets[0]]

    def call():
        return tq.verify_drafts(still[0], still[1], new, still[4], still[5], still[2], still[3] if tree else None)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for data in sets * 2:
        for a, b in zip(still, data):
            if a is not None:
                a.copy_(b)
        want = [x.clone() for x in call()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_what_python_refuses(tq):
    import torch

    counts = [3, 3]
    args = [None if x is None else x.cuda() for x in make(counts, 20, True, True, torch.float32, 1)]
    new = batch_of(tq, counts)

    def no(**kw):
        d = dict(tokens=args[0], target=args[1], new=new, accept=args[4], final=args[5], draft=args[2], parents=args[3]) | kw
        with pytest.raises(tq.InvalidArgument):
            tq.verify_drafts(**d)

    no(tokens=args[0].int()), no(tokens=args[0][:5]), no(target=args[1].double()), no(target=args[1][:5]), no(target=args[1][:, :0])
    no(draft=args[2].half()), no(draft=args[2][:, :19]), no(parents=args[3].long()), no(parents=args[3][:4]), no(accept=args[4][:3])
    no(accept=args[4].double()), no(final=args[5][:1]), no(final=args[5].cpu()), no(target=args[1].cpu()), no(tokens=args[0].cpu())
    empty = tq.KVBatch(torch.zeros(0, 1, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda(), 3)
    path, kept, token = tq.verify_drafts(args[0][:0], args[1][:0], empty, args[4][:0], args[5][:0])
    assert path.shape == (0, 3) and kept.shape == token.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("tree,draft", [(False, True), (True, False), (True, True)])
def test_padded_batches(tq, tree, draft):
    """Rows behind the last sequence, sequences of fewer rows than max_tokens, sequences of none, a batch of none at all."""
    import torch

    counts = [3, 0, 5, 1]
    tokens, p, q, parents, accept, final = make(counts, 500, tree, draft, torch.float32, 12)
    pad = lambda x, v: None if x is None else torch.cat([x, torch.full((7, *x.shape[1:]), v, dtype=x.dtype)])  # noqa: E731
    new = batch_of(tq, counts, most=9, extra=7)
    check(tq, counts, pad(tokens, 1 << 50), pad(p, float("nan")), pad(q, float("nan")), pad(parents, 0), pad(accept, float("nan")), final, not tree, new)
    none = tq.KVBatch(torch.zeros(2, 1, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda(), 0)
    e = lambda x: None if x is None else x[:0].cuda()  # noqa: E731
    path, kept, token = tq.verify_drafts(e(tokens), e(p), none, e(accept), final[:2].cuda(), e(q), e(parents) if tree else None)
    assert path.shape == (2, 0) and kept.tolist() == [0, 0] and token.tolist() == [-1, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("b,vocab", [(2500, 131072), (10000, 32768)])
def test_probabilities_past_32_bit_offsets(tq, draft, b, vocab):
    """5 GB of each model's: the last sequences are those of a call of their own."""
    import torch

    t = 8
    g = torch.Generator("cuda").manual_seed(5)
    p = torch.empty(b * t, vocab, dtype=torch.bfloat16, device="cuda").uniform_(generator=g).mul_(2.0 ** -16)
    q = torch.empty_like(p).uniform_(generator=g).mul_(2.0 ** -16) if draft else None
    tokens = torch.randint(0, vocab, (b * t,), generator=g, device="cuda")
    accept, final = torch.rand(b * t, generator=g, device="cuda") * (1 if draft else 2.0 ** -17), torch.rand(b, generator=g, device="cuda")
    full = lambda n: tq.KVBatch(torch.zeros(n, 1, dtype=torch.int32).cuda(), torch.full((n,), t, dtype=torch.int32).cuda(), t)  # noqa: E731
    for parents in (None, torch.tensor([-1, 0, 0, 1, 1, 2, 3, 3], dtype=torch.int32).repeat(b).cuda()):
        whole = tq.verify_drafts(tokens, p, full(b), accept, final, q, parents)
        for first in (0, 2 ** 31 // (t * vocab) - 1, b - 3):  # (around 2^31 elements)
            rows, seqs = slice(first * t, (first + 3) * t), slice(first, first + 3)
            part = tq.verify_drafts(tokens[rows], p[rows], full(3), accept[rows], final[seqs], None if q is None else q[rows],
                                    None if parents is None else parents[rows])
            for a, c in zip(whole, part):
                assert torch.equal(a[seqs], c)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [262144, 262145, 300001, 1100000])
def test_vocabularies_of_more_than_one_round_of_sums(tq, vocab):
    """Against sums in 64 bits on the device: the first token whose running sum passes the goal."""
    import torch

    g = torch.Generator("cuda").manual_seed(vocab)
    p = torch.softmax(torch.randn(6, vocab, generator=g, device="cuda"), 1)
    q = torch.softmax(torch.randn(6, vocab, generator=g, device="cuda"), 1)
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    accept, final = torch.ones(6, device="cuda"), torch.tensor([0.0, 0.3, 0.999], device="cuda")
    new = tq.KVBatch(torch.zeros(3, 1, dtype=torch.int32).cuda(), torch.full((3,), 2, dtype=torch.int32).cuda(), 2)
    for draft in (None, q):
        left = p[::2].double().clone()
        yes = torch.zeros(3, dtype=torch.bool, device="cuda")
        if draft is None:
            left[:, 0] = 0
        else:
            yes = q[::2, 0] < p[::2, 0]  # token 0, by a number of 1: the leaf's own probabilities follow
            left = torch.where(yes[:, None], p[1::2].double(), (left - q[::2].double()).clamp_min(0))
        sums = left.cumsum(1)
        goal = final.double()[:, None] * sums[:, -1:]
        want = (sums <= goal).sum(1)
        path, kept, token = tq.verify_drafts(tokens, p, new, accept, final, draft)
        assert torch.equal(kept, 1 + yes.int()) and torch.equal(token, want)
    # all of it beyond the first rounds
    p.zero_()
    p[:, vocab - 2] = 0.5
    assert tq.verify_drafts(tokens, p, new, accept, final)[2].tolist() == [vocab - 2] * 3
    # nothing left (q takes all): the target's own
    path, kept, token = tq.verify_drafts(tokens, p, new, accept, final, p * 2)
    assert token.tolist() == [vocab - 2] * 3
