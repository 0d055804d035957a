"""What tq_kv_read rounds: f32(code * scale), then to the type, in both of its layouts."""
import pytest

from test_gpu_cache import TYPES, dtype_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [128, 97])
def test_values_are_rounded_to_f32_first(tq, codes, dtype, d):
    """A million products of 24 and 8 (4) bits: some hundred have an f32 value halfway between two of f16, which their own
    last bits would send the other way."""
    import torch

    g = torch.Generator("cuda").manual_seed(d)
    cache = tq.KVCache.allocate(16, 64, 8, d, tq.QuantDType.Int8 if codes == "i8" else tq.QuantDType.FP8)
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if codes == "i8":
            c[..., :d] = torch.randint(-128, 128, (16, 8, 64, d), device="cuda", generator=g).to(torch.int8)
        else:
            c[..., :d] = torch.randint(0, 127, (16, 8, 64, d), device="cuda", generator=g).to(torch.uint8)
        s.copy_(torch.rand(16, 8, 64, device="cuda", generator=g) + 0.5)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    n = 16 * 64
    got = cache.read(tq.KVBatch(table, torch.tensor([n], dtype=torch.int32, device="cuda"), n), dtype_of(dtype))
    for y, c, s in zip(got, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        x = (c if codes == "i8" else c.view(torch.float8_e4m3fn)).float()[..., :d]
        want = (x * s[..., None]).transpose(1, 2).reshape(n, 8, d).to(dtype_of(dtype))
        assert torch.equal(y, want), float((y != want).double().mean())
