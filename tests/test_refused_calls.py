"""Calls that are refused are refused as such (InvalidArgument), and before anything is written."""
import pytest


@pytest.mark.gpu
def test_a_layer_that_is_refused_has_not_written_its_cache(tq):
    """Output adapters of another projection, of rows of another call or of another type, beside none for q, k and v."""
    import torch
    from test_gpu_cache import Case, rand

    h, d, rows = 2, 64, [3, 2]
    e = h * d
    layer = tq.QuantizedMultiheadAttention.from_tensors(h, *(rand(i, e, e, std=0.1) for i in range(4)), qconfig=tq.QConfig.default_int8())
    pair = lambda k, n: tq.Adapters.from_tensors([(torch.randn(8, k), torch.randn(n, 8))])  # noqa: E731
    qkv, out, index = pair(e, 3 * e), pair(e, e), torch.zeros(5, dtype=torch.int32).cuda()
    case, x = Case(tq, [20, 9], rows, 16, h, d, "i8"), rand(9, 5, e)
    before = {n: getattr(case.cache, n).clone() for n in ("k", "k_scale", "v", "v_scale")}
    for adapters, i in (((None, qkv), index), ((None, out), None), ((None, out), index[:4]), ((None, out), index.long()), ((None, out), index.cpu()),
                        ((None, pair(e + 1, e)), index), ((qkv, qkv), index), ((out, out), index), ((qkv, out), index.float())):
        with pytest.raises(tq.InvalidArgument):
            layer.forward_cached(x, case.cache, case.batch, adapters=adapters, index=i)
        for n, t in before.items():
            assert torch.equal(getattr(case.cache, n), t), n
    layer.forward_cached(x, case.cache, case.batch, adapters=(None, out), index=index)
    assert not torch.equal(case.cache.k, before["k"])


@pytest.mark.gpu
def test_adapters_of_what_is_no_tensor(tq):
    import torch

    ad = tq.Adapters.from_tensors([(torch.randn(8, 32), torch.randn(20, 8))])
    x, y, index = torch.randn(3, 32, device="cuda"), torch.randn(3, 20, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (None, 5, [1.0, 2.0], torch.zeros((), dtype=torch.int32, device="cuda"), torch.zeros(()), x.cpu().numpy()):
        for args in ((bad, index, y), (x, bad, y), (x, index, bad)) + (() if bad is None else ((x, index, y, bad),)):
            with pytest.raises(tq.InvalidArgument):
                ad.add(*args)
    want = ad.add(x, index, y)  # parameters are tensors
    p = lambda t: torch.nn.Parameter(t.clone(), requires_grad=False)  # noqa: E731
    assert torch.equal(ad.add(p(x), p(index), p(y)), want)
    out = p(torch.zeros_like(y))
    assert ad.add(x, index, y, out=out) is out and torch.equal(out, want)


@pytest.mark.gpu
def test_sizes_past_the_kernels(tq):
    """More than 2^30 tokens of a vocabulary, or rows: no workspace, and an error that says so."""
    import torch

    new = tq.KVBatch(torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int32).cuda(), 1)
    one, wide = torch.zeros(1, device="cuda"), torch.zeros(1, (1 << 30) + 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(tq.InvalidArgument):
        tq.verify_drafts(torch.zeros(1, dtype=torch.int64, device="cuda"), wide, new, one, one)
    m = (1 << 30) + 1
    ad = tq.Adapters.from_tensors([(torch.randn(8, 1), torch.randn(1, 8))])
    y = torch.zeros(m, 1, device="cuda")
    with pytest.raises(tq.InvalidArgument):
        ad.add(wide.view(m, 1), torch.zeros(m, dtype=torch.int32, device="cuda"), y, out=y)
