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
