"""QuantizedMultiheadAttention.forward_cached in every mode of its projections: the calls that it stands for, bit for bit, and
its parts against 64 bits."""
import pytest

from test_gpu_cache import Case, rand
from test_gpu_kv_attention import exact_rows, near

pytestmark = pytest.mark.gpu


def configs(tq):
    D = tq.QuantDType
    return {"w8": tq.QConfig(D.Int8, D.UInt8, True, True), "w8a8": tq.QConfig(D.Int8, D.Int8, True, True),
            "w4": tq.QConfig.default_int4(), "fp8": tq.QConfig(D.FP8, D.FP8, True, True),
            "fp8_weight": tq.QConfig(D.FP8, D.UInt8, True, True), "fp8_block": tq.QConfig.fp8_block()}


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("mode", ["w8", "w8a8", "w4", "fp8", "fp8_weight", "fp8_block"])
@pytest.mark.parametrize("lengths,new,heads,e", [([9, 40], [1, 1], 2, 256), ([30, 70, 3], [30, 17, 3], 4, 128), ([200], [90], 1, 128)])
@pytest.mark.parametrize("turned,tree", [(False, False), (True, False), (True, True)])
def test_the_layer_is_its_calls(tq, codes, mode, lengths, new, heads, e, turned, tree):
    import torch

    ws = [rand(30 + i, e, e, std=0.1) for i in range(4)]
    bias = [rand(40 + i, e, std=0.1) for i in range(4)]
    mha = tq.QuantizedMultiheadAttention.from_tensors(heads, *ws, *bias, configs(tq)[mode])
    assert mha.qkv.mode == mode
    d = e // heads
    a, b = (Case(tq, lengths, new, 16, heads, d, codes) for _ in range(2))
    for c in (a, b):
        c.fill(50)
    x = rand(51, a.rows, e)
    rot = tq.Rotary.from_base(d) if turned else None
    seen = torch.rand(a.rows, max(new), generator=torch.Generator().manual_seed(e)) < 0.5
    words = tq.tree_mask(seen).cuda() if tree else None
    got = mha.forward_cached(x, a.cache, a.batch, rot, tree=words)
    xin = x.to(torch.bfloat16) if mode == "w4" else x
    q, k, v = (t.reshape(a.rows, heads, d) for t in mha.qkv(xin).split(e, 1))
    q = b.cache.write_rotary(q, k, v, rot, b.batch) if turned else (b.cache.write(k, v, b.batch), q)[1]
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(a.cache, name), getattr(b.cache, name)), name
    o = b.cache.attention(q, b.batch, tree=words)
    if not tree:
        for i in range(len(lengths)):
            ref, pv, top, size = exact_rows(b, q, i)
            tol = 2 * 2.0 ** -24 * ((d + 16) * size + 8 * (top + 64)) * pv
            near(o[int(b.offsets[i]):int(b.offsets[i + 1])], ref.cpu(), tol.cpu())
    o = o.reshape(a.rows, e)
    assert got.shape == x.shape and got.dtype == torch.float32 and torch.isfinite(got).all()
    assert torch.equal(got, mha.out_proj(o.to(torch.bfloat16) if mode == "w4" else o))
