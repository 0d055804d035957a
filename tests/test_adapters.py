"""Low-rank adapters beside a projection (tq_adapters_add): refusals on the CPU, sums on the GPU against 64 bits."""
import ctypes
import random

import pytest

from test_cache_abi import I32, I64, PTR, refuse, structure

AdaptersDesc = structure(("a", PTR), ("b", PTR), ("scales", PTR), ("count", I64), ("parts", I64), ("rank", I64), ("k", I64), ("n", I64),
                         ("dtype", I32))
HELD = []


def at(x):
    """The address of a structure, which stays."""
    HELD.append(x)
    return None if x is None else ctypes.addressof(x)


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def desc(**kw):
    return AdaptersDesc(**(dict(a=256, b=256, scales=256, count=4, parts=2, rank=32, k=100, n=60, dtype=1) | kw))


def test_the_packed_descriptor_is_the_structure(abi):
    assert abi.adapters_desc(1, 2, 3, 4, 5, 6, 7, 8, 1) == bytes(AdaptersDesc(1, 2, 3, 4, 5, 6, 7, 8, 1))


def test_refusals(abi):
    def no(d, x=1 << 20, dtype=2, m=30, index=1 << 21, y=1 << 22, out=1 << 22, ws=256, nb=1 << 40):
        refuse(abi, "tq_adapters_add", at(d), x, dtype, m, index, y, out, ws, nb, None)

    for kw in (dict(a=None), dict(a=264), dict(b=None), dict(b=264), dict(scales=258), dict(count=0), dict(count=(1 << 20) + 1), dict(parts=0),
               dict(parts=17, n=17), dict(parts=7), dict(rank=0), dict(rank=8), dict(rank=24), dict(rank=272), dict(k=0), dict(k=(1 << 24) + 1),
               dict(n=0), dict(n=1 << 25), dict(dtype=2), dict(dtype=3), dict(dtype=-1)):
        no(desc(**kw))
        assert abi.entry("tq_adapters_workspace_bytes")(at(desc(**kw)), 3) == -1
    no(None)
    for kw in (dict(x=None), dict(x=(1 << 20) + 2), dict(dtype=3), dict(m=-1), dict(m=1 << 31), dict(index=None), dict(index=(1 << 21) + 2), dict(y=None), dict(y=(1 << 22) + 2, out=1 << 23),
               dict(out=None), dict(out=(1 << 23) + 2),
               dict(out=1 << 20), dict(out=(1 << 20) + 4 * 30 * 100 - 4), dict(out=(1 << 20) - 4 * 30 * 60 + 4), dict(out=1 << 21),
               dict(out=(1 << 21) + 4 * 29), dict(out=(1 << 22) + 4), dict(out=(1 << 22) - 4), dict(out=(1 << 22) + 4 * 30 * 60 - 4), dict(ws=None), dict(ws=264), dict(nb=100)):
        no(desc(), **kw)
    no(desc(parts=16, rank=256, n=1 << 24), m=1 << 30, nb=1 << 62)  # more blocks than a launch has
    # t of one share of K where the tiles of tokens are as many as the CUs take at once
    assert abi.entry("tq_adapters_workspace_bytes")(at(desc(rank=256)), 1 << 20) == 4 * (1 << 15) + (1 << 20) * 512 * 4
    need = abi.entry("tq_adapters_workspace_bytes")(at(desc()), 30)
    assert need >= 30 * 64 * 4 and need % 16 == 0
    assert abi.entry("tq_adapters_workspace_bytes")(at(desc()), 3) == 0 < abi.entry("tq_adapters_workspace_bytes")(at(desc(k=1 << 10)), 3)
    no(desc(), nb=need - 1)
    abi.call("tq_adapters_add", at(desc()), None, 2, 0, None, None, None, None, 0, None)
    assert abi.entry("tq_adapters_workspace_bytes")(at(desc()), 0) == 0


def made(m, count, r, parts, k, n, dtype, weights, seed, runs=False):
    """x, y, a, b, scales, index as a program has them; one row of six has no adapter."""
    import torch

    g, rng = torch.Generator("cuda").manual_seed(seed), random.Random(seed)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    index = [rng.choice([rng.randrange(count)] * 5 + [rng.choice([-1, count, -5, 1 << 30])]) for _ in range(m)]
    if runs:
        index.sort()
    return (f(m, k).to(getattr(torch, dtype)), f(m, n), (f(count, parts, r, k) * k ** -0.5).to(getattr(torch, weights)),
            (f(count, n, r) * r ** -0.5).to(getattr(torch, weights)), torch.rand(count, generator=g, device="cuda") + 0.5,
            torch.tensor(index, dtype=torch.int32).cuda())


def reference(x, y, a, b, scales, index):
    """The sums in 64 bits, and what each may be off: products are exact, and no more than 3 (K + rank) + 64 additions and
    roundings (planes, shares, the scale) of 2^-24 lie on an element's way."""
    import torch

    count, parts, r, k = a.shape
    n = b.shape[1]
    ref, size = y.double().clone(), y.double().abs()
    for i in sorted(set(index.tolist())):
        if not 0 <= i < count:
            continue
        rows = (index == i).nonzero()[:, 0]
        for p in range(parts):
            cols, s = slice(p * n // parts, (p + 1) * n // parts), 1.0 if scales is None else float(scales[i])
            t = (x[rows].double() @ a[i, p].double().t().contiguous(), x[rows].double().abs() @ a[i, p].double().abs().t().contiguous())
            ref[rows, cols] += s * (t[0] @ b[i, cols].double().t().contiguous())
            size[rows, cols] += abs(s) * (t[1] @ b[i, cols].double().abs().t().contiguous())
    return ref, size * (3 * (k + r) + 64) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["bfloat16", "float16"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,count,r,parts,k,n", [
    (1, 1, 16, 1, 64, 64), (1, 3, 1, 1, 1, 1), (17, 4, 8, 1, 100, 37), (16, 20, 16, 2, 128, 64), (65, 70, 16, 1, 72, 130), (33, 2, 64, 3, 200, 96),
    (5, 3, 128, 1, 520, 48), (40, 3, 256, 2, 64, 70), (260, 5, 16, 1, 264, 100), (300, 300, 33, 1, 64, 52), (1030, 3, 48, 3, 96, 66),
    (290, 2, 100, 1, 65, 33), (270, 2, 200, 16, 40, 64), (64, 1, 16, 1, 4097, 20), (2, 2, 16, 1, 6000, 5)])
def test_sums(tq, m, count, r, parts, k, n, dtype, weights):
    import torch

    for runs in (False, True):
        x, y, a, b, scales, index = made(m, count, r, parts, k, n, dtype, weights, 10 * m + k, runs)
        scales = scales if runs else None
        ad = tq.Adapters(a, b, scales)
        got = ad.add(x, index, y)
        ref, tol = reference(x, y, a, b, scales, index)
        err = (got.double() - ref).abs()
        assert got.dtype == torch.float32 and (err <= tol).all(), float((err / tol).max())
        none = (index < 0) | (index >= count)
        assert torch.equal(got[none], y[none])
        again = y.clone()
        assert ad.add(x, index, again, out=again) is again and torch.equal(again, got)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["bfloat16", "float16"])
@pytest.mark.parametrize("m", [3, 40, 400])
def test_every_bit_of_x_and_of_the_weights_counts(tq, m, weights):
    """One input to one rank to one output: the product of 24-bit and 8-bit (or 11-bit) numbers, exactly its f32 value where it
    has no more bits, in every place of a tile."""
    import torch

    r, k, n = 48, 200, 100
    g = torch.Generator("cuda").manual_seed(m)
    x = torch.randint(-(1 << 24) + 1, 1 << 24, (m, k), generator=g, device="cuda").float()
    a, b = torch.zeros(2, r, k), torch.zeros(2, n, r)
    pick = torch.stack([torch.randperm(k)[:r] for _ in range(2)])
    out = torch.stack([torch.randperm(n)[:r] for _ in range(2)])
    for i in range(2):
        a[i, torch.arange(r), pick[i]] = 0.5
        b[i, out[i], torch.arange(r)] = 2.0 ** 20
    index = torch.randint(0, 2, (m,), generator=g, device="cuda", dtype=torch.int32)
    ad = tq.Adapters(a.to(getattr(torch, weights)).cuda(), (b if weights == "bfloat16" else b / 64).to(getattr(torch, weights)).cuda())
    want = torch.zeros(m, n, device="cuda")
    for i in range(2):
        rows = (index == i).nonzero()[:, 0]
        want[rows[:, None], out[i].cuda()] = x[rows[:, None], pick[i].cuda()] * (2.0 ** 19 if weights == "bfloat16" else 2.0 ** 13)
    assert torch.equal(ad.add(x, index, torch.zeros(m, n, device="cuda")), want)
    # weights of all their bits times 1: an odd number of 8 (11) bits, ranks added one by one
    bits = 8 if weights == "bfloat16" else 11
    w = torch.randint(0, 1 << bits - 1, (1, r, k), generator=g, device="cuda").mul_(2).add_(1).to(getattr(torch, weights))
    one = tq.Adapters(w, torch.eye(r, dtype=w.dtype, device="cuda")[None])
    hot = torch.zeros(m, k, device="cuda")
    at_ = torch.randint(0, k, (m,), generator=g, device="cuda")
    hot[torch.arange(m, device="cuda"), at_] = 4097.0  # 13 bits: 24 in all
    got = one.add(hot, torch.zeros(m, dtype=torch.int32, device="cuda"), torch.zeros(m, r, device="cuda"))
    assert torch.equal(got, (w[0, :, at_].t().double() * 4097.0).float())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("dtype,weights", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float16")])
def test_what_a_row_does_not_use_cannot_reach_it(tq, m, dtype, weights):
    """Rows of NaN and infinities, and adapters of them: the other rows are what they were; they themselves are not finite."""
    import torch

    x, y, a, b, scales, index = made(m, 6, 24, 1, 80, 40, dtype, weights, 3)
    index = torch.where(index < 0, -1, index.clamp(-1, 6))
    ad = tq.Adapters(a, b, scales)
    want = ad.add(x, index, y)
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[1, 5, m - 1]] = True
    x2, a2, b2 = x.clone(), a.clone(), b.clone()
    x2[1], x2[5, 3], x2[m - 1, 79] = float("nan"), float("inf"), float("-inf")
    a2[2, 0, 3, 5], b2[4, 7, 1] = float("nan"), float("inf")
    got = tq.Adapters(a2, b2, scales).add(x2, index, y)
    named = (index >= 0) & (index < 6)
    touched = (bad & named) | (index == 2)
    rest = ~touched & (index != 4)
    assert torch.equal(got[rest], want[rest])
    assert not torch.isfinite(got[touched]).any(1).all() or not torch.isfinite(got[touched]).all()
    only = (index == 4) & ~bad  # one output of theirs
    cols = torch.arange(40, device="cuda") != 7
    assert torch.equal(got[only][:, cols], want[only][:, cols]) and not torch.isfinite(got[only][:, 7]).any()


@pytest.mark.gpu
def test_large_and_tiny_values(tq):
    """Near the ends of f32: planes are cut, not rounded, so nothing overflows that the sums do not."""
    import torch

    big = torch.finfo(torch.float32).max
    x = torch.zeros(4, 64, device="cuda")
    x[0, 0], x[1, 1], x[2, 2], x[3, 3] = big, -big, 2.0 ** -100, 1.1754944e-38
    a = torch.eye(16, 64, dtype=torch.bfloat16, device="cuda")[None]
    b = torch.eye(16, dtype=torch.bfloat16, device="cuda")[None]
    got = tq.Adapters(a, b).add(x, torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, 16, device="cuda"))
    assert torch.equal(got[:3], x[:3, :16]) and got[3, 3] >= 0 and abs(float(got[3, 3]) - 1.1754944e-38) <= 1.1754944e-38
    halves = torch.tensor([65504.0, 2.0 ** -24, -2.0 ** -14, 1.0009765625], device="cuda").half()
    for w, v in ((halves, torch.ones(4, device="cuda")), (torch.ones(4, device="cuda").half(), halves.float()), (halves[[1]].expand(4), halves.float())):
        a = torch.zeros(1, 4, 4, dtype=torch.float16, device="cuda")
        a[0, range(4), range(4)] = w
        got = tq.Adapters(a, torch.eye(4, device="cuda").half()[None]).add(torch.diag(v), torch.zeros(4, dtype=torch.int32, device="cuda"),
                                                                         torch.zeros(4, 4, device="cuda"))
        assert torch.equal(got, torch.diag(w.float() * v))


@pytest.mark.gpu
def test_adapters_of_many_ranks_and_strided_tensors(tq):
    import torch

    g = torch.Generator("cuda").manual_seed(1)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    pairs = [(f(r, 72), f(40, r)) for r in (1, 16, 37, 200)]
    ad = tq.Adapters.from_tensors(pairs, [1.0, 2.0, 0.5, 1.5])
    x, y, index = f(50, 72), f(50, 40), torch.arange(50, dtype=torch.int32, device="cuda") % 5
    got = ad.add(x, index, y)
    for i, (a, b) in enumerate(pairs):
        ref, tol = reference(x, y, a.bfloat16()[None, None], b.bfloat16()[None], torch.tensor([1.0, 2.0, 0.5, 1.5][i:i + 1]),
                             torch.where(index == i, 0, -1))
        assert ((got.double() - ref).abs() <= tol)[index == i].all()
    assert torch.equal(got[index == 4], y[index == 4])
    wide = f(50, 144)[:, ::2]
    assert torch.equal(ad.add(wide, index, y), ad.add(wide.contiguous(), index, y))
    odd = torch.empty(50 * 72 + 1, device="cuda")[1:].view(50, 72)  # rows off 16 bytes: element by element
    odd.copy_(x)
    assert torch.equal(ad.add(odd, index, y), got)
    shifted = torch.empty(50 * 40 + 1, device="cuda")[1:].view(50, 40)
    shifted.copy_(y)
    assert torch.equal(ad.add(x, index, shifted), got)
    for part in ([1, 2], [2, 1]):  # slices of a larger stack
        sl = tq.Adapters(ad.a.new_zeros(4, 3, 16, 64)[part[0]:part[0] + part[1]], ad.b.new_ones(4, 30, 16)[part[0]:part[0] + part[1]])
        assert sl.count == part[1] and sl.parts == 3
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        side = ad.add(x, index, y)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(side, got)
    # no rows; an empty projection is refused
    assert ad.add(x[:0], index[:0], y[:0]).shape == (0, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 500])
def test_captured_and_replayed(tq, m):
    import torch

    x, y, a, b, scales, index = made(m, 4, 16, 2, 128, 64, "float32", "bfloat16", 4)
    ad, s = tq.Adapters(a, b, scales), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ad.add(x, index, y)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ad.add(x, index, y)
    for i in range(5):
        x.normal_(), y.normal_()
        index.copy_(index.roll(1))
        want = ad.add(x, index, y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


MODES = ["w8", "w8a8", "w4", "fp8", "fp8_weight", "fp8_block"]


def config(tq, mode):
    D, Q = tq.QuantDType, tq.QConfig
    return {"w8": Q.default_int8(), "w8a8": Q(D.Int8, D.Int8, True, True), "w4": Q.default_int4(), "fp8": Q(D.FP8, D.FP8, True, True),
            "fp8_weight": Q(D.FP8, D.Int8, True, True), "fp8_block": Q.fp8_block()}[mode]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m", [1, 6, 70])
def test_a_quantized_linear_with_adapters_is_its_two_calls(tq, mode, m):
    import torch

    x, _, a, b, scales, index = made(m, 3, 8, 1, 256, 128, "bfloat16" if mode == "w4" else "float32", "bfloat16", m)
    lin = tq.QuantizedLinear.from_tensors(torch.randn(128, 256, device="cuda") * 0.05, torch.randn(128, device="cuda"), config(tq, mode))
    assert lin.mode == mode
    ad = tq.Adapters(a, b, scales)
    want = ad.add(x, index, lin(x))
    assert torch.equal(lin(x, ad, index), want) and torch.equal(lin.forward(x, adapters=ad, index=index), want)
    if m == 1:
        assert torch.equal(lin(x[0], ad, index), want[0])
    for bad in (index[:0], None, torch.zeros(m + 1, dtype=torch.int32, device="cuda")):
        with pytest.raises(tq.InvalidArgument):
            lin(x, ad, bad)
    other = tq.QuantizedLinear.from_tensors(torch.randn(64, 256, device="cuda"), None, config(tq, mode))
    with pytest.raises(tq.InvalidArgument):
        other(x, ad, index)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["w8a8", "w4", "fp8_block"])
def test_the_attention_layer_over_a_cache_with_adapters_is_its_calls(tq, mode):
    """Requests' own adapters on q, k and v and on the output, positions of several axes, a drafted tree."""
    import torch
    from test_gpu_cache import Case, rand

    h, d, rows = 2, 64, [5, 5]
    e = h * d
    w = [rand(i, e, e, std=0.1) for i in range(4)]
    layer = tq.QuantizedMultiheadAttention.from_tensors(h, *w, qconfig=config(tq, mode))
    _, _, a, b, scales, _ = made(1, 3, 8, 3, e, 3 * e, "float32", "bfloat16", 5)
    _, _, a2, b2, _, _ = made(1, 3, 16, 1, e, e, "float32", "bfloat16", 6)
    qkv, out = tq.Adapters(a, b, scales), tq.Adapters(a2, b2)
    index = torch.tensor([2] * 5 + [0] * 4 + [-1], dtype=torch.int32).cuda()
    x, rot = rand(9, 10, e), tq.Rotary.from_base(d, axes=tq.Rotary.axes_in_blocks([8, 12, 12]))
    pos = torch.randint(0, 50, (3, 10), device="cuda")
    one, two = (Case(tq, [20, 9], rows, 16, h, d, "i8") for _ in range(2))
    got = layer.forward_cached(x, one.cache, one.batch, rot, pos, adapters=(qkv, out), index=index)
    y = layer.qkv(layer._act(x), qkv, index)
    q, k, v = (y[:, i * e:(i + 1) * e].view(10, h, d) for i in range(3))
    o = two.cache.attention(two.cache.write_rotary(q, k, v, rot, two.batch, pos), two.batch).view(10, e)
    assert torch.equal(got, layer.out_proj(layer._act(o), out, index))
    assert torch.equal(one.cache.k, two.cache.k) and torch.equal(one.cache.v, two.cache.v)
    assert not torch.equal(got, layer.forward_cached(x, two.cache, two.batch, rot, pos))
    layer.forward_cached(x, two.cache, two.batch, rot, pos, adapters=(qkv, out), index=torch.full_like(index, -1))
    plain = layer.forward_cached(x, one.cache, one.batch, rot, pos)
    assert torch.equal(plain, layer.forward_cached(x, two.cache, two.batch, rot, pos, adapters=(None, out), index=torch.full_like(index, -1)))


@pytest.mark.gpu
def test_what_python_refuses(tq):
    import torch

    x, y, a, b, scales, index = made(4, 3, 8, 2, 32, 20, "float32", "bfloat16", 1)
    for args in ((a.float(), b), (a, b.half()), (a[:2], b), (a, b[:, :, :7]), (a, b[:, :19]), (a[0, 0], b), (a, b, scales[:2]), (a, b, scales.half()),
                 (a.cpu(), b), (a[:, :, :0], b[..., :0]), (a[:0], b[:0]), (a.new_zeros(1, 1, 257, 8), b.new_zeros(1, 4, 257))):
        with pytest.raises(tq.InvalidArgument):
            tq.Adapters(*args)
    ad = tq.Adapters(a, b, scales)
    with pytest.raises(AttributeError):
        ad.a = a
    for args in ((x.double(), index, y), (x[:3], index, y), (x[:, :31], index, y), (x, index.long(), y), (x, index[:2], y), (x, index, y.half()),
                 (x, index, y[:, :19]), (x, index, y.t().contiguous().t()), (x.cpu(), index, y), (x, index.cpu(), y), (x, index, y.cpu()),
                 (x, index, y, y.half()), (x, index, y, y[:2]), (x, index, y, torch.as_strided(x, (4, 20), (20, 1)))):
        with pytest.raises(tq.InvalidArgument):
            ad.add(*args)
    with pytest.raises(tq.InvalidArgument):
        tq.Adapters.from_tensors([])
    with pytest.raises(tq.InvalidArgument):
        tq.Adapters.from_tensors([(a[0, 0], b[0]), (a[0, 0, :, :30], b[0])])


@pytest.mark.gpu
def test_outputs_and_inputs_past_32_bit_offsets(tq):
    """9 GB of outputs, 5 GB of inputs: rows about each 2^31st element are those of a call of their own."""
    import torch

    for m, k, n, dtype in ((70000, 16, 32768, torch.float32), (300000, 8192, 16, torch.bfloat16)):
        g = torch.Generator("cuda").manual_seed(3)
        x = torch.empty(m, k, dtype=dtype, device="cuda").normal_(generator=g)
        y = torch.empty(m, n, device="cuda").normal_(generator=g)
        a = (torch.randn(3, 16, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
        b = torch.randn(3, n, 16, generator=g, device="cuda").bfloat16()
        ad = tq.Adapters(a, b)
        index = torch.randint(-1, 3, (m,), generator=g, device="cuda", dtype=torch.int32)
        width = max(k, n)
        rows = sorted({0, m - 40, max((1 << 31) // width - 20, 0), max((1 << 32) // width - 20, 0)} & set(range(m - 39)))
        before = [y[r:r + 40].clone() for r in rows]
        ad.add(x, index, y, out=y)
        for r, part in zip(rows, before):
            ref, tol = reference(x[r:r + 40], part, a[:, None], b, None, index[r:r + 40])
            assert ((y[r:r + 40].double() - ref).abs() <= tol).all(), r


@pytest.mark.gpu
def test_two_streams_at_once(tq):
    import torch

    cases = [made(m, 5, 16, 1, 512, 1024, "float32", "bfloat16", m) for m in (7, 600)]
    ads = [tq.Adapters(a, b, scales) for _, _, a, b, scales, _ in cases]
    want = [ad.add(x, index, y) for ad, (x, y, _, _, _, index) in zip(ads, cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (ad, (x, y, _, _, _, index)) in enumerate(zip(ads, cases)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ad.add(x, index, y))
    torch.cuda.synchronize()
    for w, all_ in zip(want, got):
        assert all(torch.equal(w, z) for z in all_)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,r", [(2049, 64, 16), (2048, 64, 16), (2100, 4100, 16), (3900, 4100, 16), (3100, 4100, 32), (513, 2048, 40), (600, 2000, 70), (400, 2100, 130), (1100, 1000, 200)])
def test_sizes_on_both_sides_of_every_form(tq, m, n, r):
    """Tiles of 16 and 32 tokens, the forms of few and many rows, each with one adapter, a few in runs and many mixed."""
    import torch

    for count, runs in ((1, True), (3, True), (50, False)):
        x, y, a, b, scales, index = made(m, count, r, 1, 130, n, "float32", "bfloat16", m + count, runs)
        ref, tol = reference(x, y, a, b, scales, index)
        assert ((tq.Adapters(a, b, scales).add(x, index, y).double() - ref).abs() <= tol).all()
    index.fill_(-1)
    assert torch.equal(tq.Adapters(a, b, scales).add(x, index, y), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,weights", [("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"), ("float16", "float16"),
                                           ("float16", "bfloat16"), ("bfloat16", "float16")])
@pytest.mark.parametrize("m,count,r,parts,k,n", [(20000, 7, 16, 1, 2601, 40), (10001, 3, 30, 1, 2600, 66), (5000, 60, 40, 1, 3500, 100),
                                                 (1100, 4, 48, 16, 1000, 64), (300, 5, 256, 16, 701, 32)])
def test_long_first_products(tq, m, count, r, parts, k, n, dtype, weights):
    """Tiles of 32 tokens, of all ranks."""
    ranks = parts * ((r + 15) // 16 * 16)
    assert m * ranks * k >= 3 << 28
    for runs in (False, True):
        x, y, a, b, scales, index = made(m, count, r, parts, k, n, dtype, weights, m + runs, runs)
        ref, tol = reference(x, y, a, b, scales, index)
        assert ((tq.Adapters(a, b, scales).add(x, index, y).double() - ref).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("count,parts,rank,k", [(1, 1, 1, 1), (3, 2, 16, 64), (2, 3, 17, 100), (5, 1, 256, 65), (1, 16, 8, 4097)])
def test_the_tiles_of_a(tq, count, parts, rank, k):
    import torch

    a = torch.randn(count, parts, rank, k, device="cuda").bfloat16()
    ranks, row = (rank + 15) // 16 * 16, (k + 63) // 64 * 64
    full = torch.zeros(count, parts, ranks, row, dtype=a.dtype, device="cuda")
    full[:, :, :rank, :k] = a
    held = tq.Adapters(a, torch.zeros(count, parts, rank, dtype=a.dtype, device="cuda")).a
    assert torch.equal(held, full.view(count, parts * ranks // 16, 16, row // 32, 32).transpose(2, 3))
    back = torch.randn(count, rank, parts, k, device="cuda").half().transpose(1, 2)  # strided, f16
    held = tq.Adapters(back, torch.zeros(count, parts, rank, dtype=torch.float16, device="cuda")).a
    full = torch.zeros(count, parts, ranks, row, dtype=torch.float16, device="cuda")
    full[:, :, :rank, :k] = back
    assert torch.equal(held, full.view(count, parts * ranks // 16, 16, row // 32, 32).transpose(2, 3))


def test_repacking_refusals(abi):
    for args in ((None, 2, 16, 64, 256), (257, 2, 16, 64, 256), (256, 2, 16, 64, None), (256, 2, 16, 64, 264), (256, -1, 16, 64, 256),
                 (256, 2, 0, 64, 256), (256, 2, 257, 64, 256), (256, 2, 16, 0, 256), (256, 2, 16, 1 << 25, 256), (256, 1 << 30, 16, 64, 256)):
        refuse(abi, "tq_repack_adapters_tiled", *args, None)
    abi.call("tq_repack_adapters_tiled", None, 0, 16, 64, None, None)
