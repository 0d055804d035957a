"""Frequencies of Rotary.from_base against the published scalings, written out plane by plane."""
import math

import pytest

pytestmark = pytest.mark.gpu


def planes(r, base, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """Angles per position: base^(-2 i / r); linear: divided by the factor; ntk: of the base that divides the slowest plane's angle
    by the factor and leaves the fastest; yarn: by the turns that a plane makes over the original length, kept from `fast` on,
    divided by the factor up to `slow`, and between them a ramp over the plane's number."""
    out = []
    if scaling == "ntk":
        base = base * factor ** (r / (r - 2.0))

    def number(turns):  # i for which original * base^(-2 i / r) / (2 pi) = turns
        return r / 2.0 * math.log(original / (2 * math.pi * turns), base)

    for i in range(r // 2):
        f = base ** (-2.0 * i / r)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            lo, hi = max(0, math.floor(number(fast))), min(r - 1, math.ceil(number(slow)))
            keep = 1.0 if i <= lo else 0.0 if i >= hi else 1.0 - (i - lo) / (hi - lo)
            f = keep * f + (1.0 - keep) * f / factor
        out.append(f)
    return out


@pytest.mark.parametrize("r,base,kw", [
    (128, 10000.0, {}), (2, 10000.0, {}), (0, 10000.0, {}), (64, 500000.0, dict(scaling="linear", factor=8.0)),
    (128, 10000.0, dict(scaling="ntk", factor=4.0)), (6, 100.0, dict(scaling="ntk", factor=2.5)),
    (128, 10000.0, dict(scaling="yarn", factor=32.0, original=4096)), (64, 150000.0, dict(scaling="yarn", factor=8.0, original=32768)),
    (128, 10000.0, dict(scaling="yarn", factor=4.0, original=4096, fast=16.0, slow=2.0)),
    (8, 10000.0, dict(scaling="yarn", factor=2.0, original=64))])
def test_frequencies(tq, r, base, kw):
    import torch

    names = {"original": "original_length", "fast": "fast_turns", "slow": "slow_turns"}
    rot = tq.Rotary.from_base(r, base, **{names.get(k, k): v for k, v in kw.items()})
    want = torch.tensor(planes(r, base, **kw), dtype=torch.float64)
    got = rot.frequencies.cpu()
    assert got.dtype == torch.float64 and got.shape == want.shape
    assert ((got - want).abs() <= 1e-12 * want).all()  # powers and logarithms in 64 bits: some hundred units of 2^-53
    assert rot.scale == (0.1 * math.log(kw["factor"]) + 1.0 if kw.get("scaling") == "yarn" else 1.0)
    if kw.get("scaling") == "ntk":
        plain = planes(r, base)
        assert got[0] == plain[0] and abs(float(got[-1]) * kw["factor"] / plain[-1] - 1.0) < 1e-12


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("d,r,pairs", [(128, 128, False), (97, 56, False), (100, 50, True), (64, 64, True), (80, 36, False)])
@pytest.mark.parametrize("far", [1 << 20, 1 << 40])
def test_a_far_token_is_turned_alike_by_every_call(tq, dtype, d, r, pairs, far):
    """A token's angles are the same numbers in calls of one token and of many, of q and k alone and with the cache, in
    every element type and layout: the f32 values that are rounded or coded are bit for bit the same."""
    import torch

    from test_gpu_cache import Case, dtype_of, rand

    n, h = 200, 3
    x = rand(d, n, h, d, dtype=dtype_of(dtype))
    rot = tq.Rotary.from_base(r, 1000.0, pairs, scale=1.25)
    pos = torch.randint(0, far, (n,), generator=torch.Generator().manual_seed(r)).cuda()
    want = rot.apply(x.float(), None, pos)[0]
    odd = torch.empty(n * (h * d + 1) + 1, device="cuda")[1:].view(n, -1)[:, :h * d].view(n, h, d)
    odd.copy_(x)
    assert torch.equal(rot.apply(odd, None, pos)[0], want)  # the same values by elements
    assert torch.equal(rot.apply(x, None, pos)[0], want.to(x.dtype))
    for i in range(0, n, 17):
        assert torch.equal(rot.apply(x[i:i + 1], None, pos[i:i + 1])[0], want[i:i + 1].to(x.dtype))
    a, b, c = (Case(tq, [n], [n], 16, h, d, "fp8") for _ in range(3))
    b.cache.write(want, x.float(), b.batch)
    assert torch.equal(a.cache.write_rotary(x, x, x, rot, a.batch, pos), want.to(x.dtype))
    for i in range(n):
        one = tq.KVBatch(c.table, torch.tensor([i + 1], dtype=torch.int32).cuda(), 1)
        part = slice(i, i + 1)
        assert torch.equal(c.cache.write_rotary(x[part], x[part], x[part], rot, one, pos[part]), want[part].to(x.dtype))
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(a.cache, name), getattr(b.cache, name)), name
        assert torch.equal(getattr(c.cache, name), getattr(b.cache, name)), name
