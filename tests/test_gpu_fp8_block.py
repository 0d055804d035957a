"""GPU parity: FP8 with a scale for each block of 128 (tq_quantize_fp8_block, tq_quantize_fp8_g128,
tq_gemm_fp8_block, tq_linear_fp8_block) against the definition in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SHAPES = [  # m, n, k
    (1, 128, 128), (1, 1, 1), (3, 5, 7), (1, 4096, 4096), (2, 130, 129), (4, 1003, 1000), (5, 16, 4000), (16, 256, 512),
    (17, 4104, 272), (31, 100, 2048), (33, 384, 1152), (64, 1000, 136), (77, 1003, 1000), (130, 520, 4000), (200, 129, 4097),
    (257, 264, 392), (513, 640, 400), (1030, 1160, 1104), (2047, 512, 640), (8, 64, 16384), (3, 72, 12304)]


def rand(seed, *shape, std=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype or torch.float32)


def e4m3(codes):
    import torch

    return codes.view(torch.float8_e4m3fn).to(torch.float32).double()


def blocks(x, rows):
    """[ceil(M / rows), rows, ceil(K / 128), 128] of [M, K], NaN where nothing lies."""
    import torch

    m, k = x.shape
    mb, kb = (m + rows - 1) // rows, (k + 127) // 128
    full = torch.full((mb * rows, kb * 128), float("nan"), dtype=x.dtype, device=x.device)
    full[:m, :k] = x
    return full.view(mb, rows, kb, 128)


def coded(x, rows):
    """Scales [.., ..] and codes of the definition: absmax over what is not NaN (infinity where nothing
    is), an f32 scale, the f32 quotient to the nearest e4m3."""
    import torch

    b = blocks(x.float(), rows)
    top = torch.where(torch.isnan(b), -torch.inf, b.abs()).amax((1, 3))
    top = torch.where(top == -torch.inf, torch.inf, top)
    s = (top.double() / 448.0).clamp_min(1e-10).float()
    q = b / s[:, None, :, None]
    c = q.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    c = torch.where(torch.isnan(q), torch.full_like(c, 0x7F), c)
    m, k = x.shape
    return s, c.reshape(b.shape[0] * rows, -1)[:m, :k]


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 130), (300, 1000), (7, 4100), (1000, 5)])
def test_weight_blocks(tq, n, k):
    import torch

    w = rand(n + k, n, k, std=0.02)
    if n > 6:
        w[2, 3] = float("nan")
        w[5, k - 1] = 0.5
        w[6, 0] = float("inf")
    q, s = tq.quantize_fp8_block(w)
    rs, rq = coded(w, 128)
    assert torch.equal(s, rs) and torch.equal(q, rq)
    back = tq.dequantize_fp8_block(q, s)
    grown = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref = (e4m3(q) * grown.double()).float()
    assert torch.equal(torch.isnan(back), torch.isnan(ref)) and torch.equal(torch.nan_to_num(back), torch.nan_to_num(ref))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 130), (17, 1000), (2, 4100), (300, 264)])
def test_activation_rows(tq, m, k, dtype):
    import torch

    x = rand(m * k, m, k, dtype=getattr(torch, dtype))
    x[m - 1, k - 1] = float("nan")
    if m > 2:
        x[1] = 0.0
    q, s = tq.quantize_fp8_g128(x)
    rs, rq = coded(x, 1)
    assert torch.equal(s, rs.t().contiguous()) and torch.equal(q[:, :k], rq) and (q[:, k:] == 0).all()


def product(qa, sa, qw, sw, bias):
    """The definition in 64 bits and its sums of absolute terms."""
    import torch

    n, k = qw.shape
    m = qa.shape[0]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(y)
    for b in range(sa.shape[0]):
        a, w = e4m3(qa[:, b * 128:min(k, b * 128 + 128)]), e4m3(qw[:, b * 128:b * 128 + 128])
        f = sa[b].double()[:, None] * sw[:, b].double().repeat_interleave(128)[:n][None]
        y += f * (a @ w.t().contiguous())
        size += f * (a.abs() @ w.abs().t().contiguous())
    if bias is not None:
        y += bias.double()
        size += bias.double().abs()
    return y, size


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_product(tq, m, n, k, bias):
    """Within what f32 sums allow: a block's at most 128 roundings of its absolute terms, the scale's
    product and each of the ceil(K / 128) blocks' additions one of the running sum."""
    import torch

    x, w = rand(m, m, k), rand(n, n, k, std=0.02)
    x[:, ::7] *= 100.0  # columns far above the rest
    b = rand(3, n, std=0.1) if bias else None
    qa, sa = tq.quantize_fp8_g128(x)
    qw, sw = tq.quantize_fp8_block(w)
    ref, size = product(qa, sa, qw, sw, b)
    got = tq.gemm_fp8_block(qa, sa, qw, sw, b)
    assert got.shape == (m, n) and got.dtype == torch.float32
    off = (got.double() - ref).abs()
    assert (off <= (min(k, 128) + 3 + (k + 127) // 128) * 2.0 ** -24 * size).all(), float((off / size).max())
    assert float(off.norm() / ref.norm()) < 1e-6
    lin = tq.QuantizedLinear("fp8_block", k, n, qw, sw, b)
    assert torch.equal(lin(x), got)
    assert torch.equal(lin(x[0]), tq.gemm_fp8_block(*tq.quantize_fp8_g128(x[:1]), qw, sw, b)[0])
    for dt in (torch.bfloat16, torch.float16):
        h = x.to(dt)
        assert torch.equal(lin(h), tq.gemm_fp8_block(*tq.quantize_fp8_g128(h), qw, sw, b))


@pytest.mark.parametrize("m,n,k,shift", [
    (1, 9001, 144, 0), (7, 16400, 257, 0), (16, 4100, 1050, 0), (16, 4097, 130, 1),  # rows after rows in a block
    (4, 48, 4096, 0), (5, 48, 4096, 0), (6, 64, 4096, 5), (2, 33, 8192, 0), (12, 20, 2176, 3),  # codes made or copied or read
    (17, 4096, 4096, 0), (32, 300, 4096, 0), (32, 4112, 512, 0), (24, 40, 4224, 0), (29, 77, 128, 7), (32, 16, 127, 0),
    (63, 500, 528, 0), (64, 130, 528, 0), (64, 130, 528, 8), (100, 260, 2048, 3), (128, 128, 4096, 0),
    (140, 260, 4112, 0), (1200, 8000, 144, 0), (2000, 4500, 784, 0),  # shares of K, with and without whole rounds before
    (100, 260, 2047, 0), (300, 500, 129, 0), (64, 128, 143, 1), (2000, 4500, 777, 5), (65, 3, 128, 9), (129, 257, 4090, 0)])
def test_product_at_its_turns(tq, m, n, k, shift):
    """Sizes beside each choice of kernel, and weights off their boundary: the bound of `test_product`."""
    import torch

    x, w, b = rand(m, m, k, dtype=torch.bfloat16), rand(n, n, k, std=0.02), rand(4, n)
    qa, sa = tq.quantize_fp8_g128(x)
    qw, sw = tq.quantize_fp8_block(w)
    if shift:
        qw = torch.full((n * k + 64,), 0x7F, dtype=torch.uint8, device="cuda")[shift:shift + n * k].view(n, k).copy_(qw)
    ref, size = product(qa, sa, qw, sw, b)
    got = tq.gemm_fp8_block(qa, sa, qw, sw, b)
    off = (got.double() - ref).abs()
    assert (off <= (min(k, 128) + 3 + (k + 127) // 128) * 2.0 ** -24 * size).all(), float((off / size).max())
    assert torch.equal(tq.QuantizedLinear("fp8_block", k, n, qw, sw, b)(x), got)


def test_weights_at_any_address(tq):
    """Weight rows that start off every boundary, and a guard behind the last row that stays unread in
    the result."""
    import torch

    m, n, k = 5, 40, 200
    x, w = rand(1, m, k), rand(2, n, k)
    qa, sa = tq.quantize_fp8_g128(x)
    qw, sw = tq.quantize_fp8_block(w)
    want = tq.gemm_fp8_block(qa, sa, qw, sw)
    for shift in (1, 2, 3, 7, 8):
        buf = torch.full((n * k + 64,), 0x7F, dtype=torch.uint8, device="cuda")
        view = buf[shift:shift + n * k].view(n, k)
        view.copy_(qw)
        assert torch.equal(tq.gemm_fp8_block(qa, sa, view, sw), want)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_nan_and_infinite_rows_stay_in_their_rows(tq, m):
    import torch

    n, k = 192, 400
    x = rand(5, m, k)
    lin = tq.QuantizedLinear.from_tensors(rand(6, n, k), None, tq.QConfig.fp8_block())
    clean = lin(x)
    bad = x.clone()
    bad[0, 399] = float("nan")
    if m > 2:
        bad[1, 0] = float("inf")
    y = lin(bad)
    assert torch.isnan(y[0]).all()
    if m > 2:
        assert torch.isnan(y[1]).all()
        assert torch.equal(y[2:], clean[2:])


@pytest.mark.parametrize("m", [1, 3, 20, 40, 100])
@pytest.mark.parametrize("k", [128, 200, 1000, 2047, 4096])
def test_nan_weights_stay_in_their_rows(tq, m, k):
    """A NaN code reaches its own output column: not the ones before and behind it, whose bytes its row's ends touch."""
    import torch

    n = 160
    x = rand(7, m, k)
    qa, sa = tq.quantize_fp8_g128(x)
    qw, sw = tq.quantize_fp8_block(rand(8, n, k))
    clean = tq.gemm_fp8_block(qa, sa, qw, sw)
    bad = qw.clone()
    bad[5, 0], bad[9, k - 1], bad[n - 1, k - 1] = 0x7F, 0xFF, 0x7F
    y = tq.gemm_fp8_block(qa, sa, bad, sw)
    hit = torch.zeros(n, dtype=torch.bool, device="cuda")
    hit[[5, 9, n - 1]] = True
    assert torch.isnan(y[:, hit]).all() and torch.equal(y[:, ~hit], clean[:, ~hit])


def test_refusals(tq):
    import torch

    qa, sa = tq.quantize_fp8_g128(rand(1, 3, 200))
    qw, sw = tq.quantize_fp8_block(rand(2, 40, 200))
    for args in ((qa[:, :200], sa, qw, sw), (qa, sa.t(), qw, sw), (qa, sa, qw, sw[:, :1]), (qa, sa, qw[:, :100], sw),
                 (qa, sa, qw, sw, torch.zeros(3, device="cuda")), (qa.float(), sa, qw, sw), (qa, sa.double(), qw, sw)):
        with pytest.raises(tq.InvalidArgument):
            tq.gemm_fp8_block(*args)
    with pytest.raises(tq.InvalidArgument):
        tq.QuantizedLinear("fp8_block", 200, 40, qw, sw[0])
    with pytest.raises(tq.InvalidArgument):
        tq.QuantizedLinear("fp8_block", 200, 40, qw, sw)(torch.zeros(2, 201, device="cuda"))
    with pytest.raises(tq.InvalidArgument):
        tq.quantize_fp8_g128(torch.zeros(2, 3, dtype=torch.float64))
    assert tq.QuantizedLinear("fp8_block", 200, 40, qw, sw)(torch.zeros(0, 200, device="cuda")).shape == (0, 40)


def test_checkpoint_and_layer(tq):
    """Saved and loaded modules give the same bits; an attention layer in this mode over a cache equals its parts."""
    import torch

    lin = tq.QuantizedLinear.from_tensors(rand(1, 300, 200, std=0.05), rand(2, 300), tq.QConfig.fp8_block())
    e, h = 256, 4
    mha = tq.QuantizedMultiheadAttention.from_tensors(h, *(rand(3 + i, e, e, std=0.06) for i in range(4)),
                                                      qconfig=tq.QConfig.fp8_block())
    back = tq.load_quantized(tq.save_quantized({"a": lin, "m": mha}))
    x = rand(9, 6, 200)
    assert torch.equal(back["a"](x), lin(x))
    y = rand(10, 2, 5, e)
    assert torch.equal(back["m"](y), mha(y))
    cache = tq.KVCache.allocate(4, 16, h, e // h, tq.QuantDType.FP8)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32).cuda()
    rot = tq.Rotary.from_base(e // h)
    flat = y.reshape(10, e)
    new = tq.KVBatch(table, torch.tensor([5, 5], dtype=torch.int32).cuda(), 5)
    got = mha.forward_cached(flat, cache, new, rot)
    q, k, v = (t.reshape(10, h, e // h) for t in mha.qkv(flat).split(e, 1))
    other = tq.KVCache.allocate(4, 16, h, e // h, tq.QuantDType.FP8)
    o = other.attention(other.write_rotary(q, k, v, rot, new), new)
    assert torch.equal(got, mha.out_proj(o.reshape(10, e)))
    # without positions the layer over the cache is its causal self over keys and values as stored
    plain = mha.forward_cached(flat, cache, new)
    kk, vv = (t.reshape(2, 5, e) for t in cache.read(new))
    full = mha._attend(q.reshape(10, e).contiguous(), kk.reshape(10, e).contiguous(), vv.reshape(10, e).contiguous(), e, e, e, 2, 5,
                       torch.triu(torch.full((1, 5, 5), float("-inf"), device="cuda"), 1))
    o = cache.attention(q, new).view(10, e)
    assert torch.equal(plain, mha.out_proj(o))
    assert ((o - full).abs() <= 1e-4 + 1e-3 * full.abs()).all()  # the attention core's own tolerance


def test_graph_replays(tq):
    import torch

    lin = tq.QuantizedLinear.from_tensors(rand(1, 512, 1024, std=0.05), None, tq.QConfig.fp8_block())
    xs = [rand(20 + i, 70, 1024) for i in range(4)]
    want = [lin(x) for x in xs]
    buf = xs[0].clone()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        lin(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lin(buf)
    for x, y in zip(xs, want):
        buf.copy_(x)
        graph.replay()
        assert torch.equal(out, y)
        lin(xs[3])
        torch.cuda.synchronize()


def test_weights_past_32_bits(tq):
    """A weight of more than 2^31 codes: its last rows give what they give alone."""
    import torch

    n, k = 140032, 16400
    g = torch.Generator(device="cuda").manual_seed(5)
    qw = torch.randint(0, 0x70, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    sw = torch.rand((n + 127) // 128, (k + 127) // 128, generator=g, device="cuda") + 0.5
    part = slice(n - 256, n)
    for m in (1, 20, 70):
        qa, sa = tq.quantize_fp8_g128(rand(6, m, k))
        y = tq.gemm_fp8_block(qa, sa, qw, sw)[:, part]
        ref, size = product(qa, sa, qw[part], sw[-2:], None)
        assert ((y.double() - ref).abs() <= (131 + (k + 127) // 128) * 2.0 ** -24 * size).all()
