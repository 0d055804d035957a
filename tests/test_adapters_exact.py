"""Low-rank adapters beside a projection: every bit of both operands of both products, in every form, and what infinities
and NaN do to the rows that use them."""
import pytest

# rows, rank, inputs, outputs: one launch; few rows in two; many rows in tiles of 16, and (rows x ranks x K from 3 2^28 on) of
# 32 tokens, each with the second product's form of few rows (few outputs, or off 4) and that of many, of every count of ranks
SIZES = [(3, 32, 100, 60), (16, 16, 250, 37), (40, 48, 200, 100), (400, 48, 200, 100), (1540, 64, 130, 1024), (700, 128, 130, 1128),
         (12300, 16, 4100, 1024), (12300, 32, 2100, 1024), (4100, 64, 3100, 400), (4100, 48, 4100, 77), (2060, 128, 3100, 400),
         (1030, 256, 3100, 800)]


def odd(g, bits, shape, dtype):
    """Numbers of just so many bits, the last one set: in [1, 2), of either sign."""
    import torch

    v = torch.randint(1 << bits - 1, 1 << bits, shape, generator=g, device="cuda") | 1
    return (v.double() * 2.0 ** (1 - bits) * (1 - 2 * torch.randint(0, 2, shape, generator=g, device="cuda"))).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["bfloat16", "float16"])
@pytest.mark.parametrize("m,r,k,n", SIZES)
def test_products_have_every_bit_of_both_operands(tq, m, r, k, n, weights):
    """One input to each rank and one rank to each output, so that an output is one product: of x (24 bits) and a, or of
    t = x and b (8 or 11 bits each).  Cut into planes whose pairs are exact and whose sums' last addition alone rounds at
    the result's size, by half a step, 2^-24 of it; those before it round what is 2^-6 of it or less.  Twice the half step is allowed.
    x without its third plane, or without its product with a's second, is off by up to 2^-15 and 2^-22."""
    import torch

    dtype, bits = getattr(torch, weights), 8 if weights == "bfloat16" else 11
    g = torch.Generator("cuda").manual_seed(m + r)
    x = odd(g, 24, (m, k), torch.float32)
    index = torch.arange(m, device="cuda", dtype=torch.int32) * 2 // m
    pick = torch.stack([torch.randperm(k, generator=g, device="cuda")[:r] for _ in range(2)])
    via = (torch.arange(n, device="cuda") * 7 + 3) % r  # an output's rank
    rank, out = torch.arange(r, device="cuda"), torch.arange(n, device="cuda")
    for first in (True, False):
        w = odd(g, bits, (2, r) if first else (2, n), dtype)
        a, b = torch.zeros(2, 1, r, k, dtype=dtype, device="cuda"), torch.zeros(2, n, r, dtype=dtype, device="cuda")
        for i in range(2):
            a[i, 0, rank, pick[i]] = w[i] if first else 1.0
            b[i, out, via] = 1.0 if first else w[i]
        got = tq.Adapters(a, b).add(x, index, torch.zeros(m, n, device="cuda"))
        for i in range(2):
            rows = (index == i).nonzero()[:, 0]
            want = x[rows][:, pick[i]].double()[:, via] * (w[i].double()[via] if first else w[i].double())
            err = ((got[rows].double() - want) / want).abs().max()
            assert err <= 2.0 ** -23, (first, i, float(err * 2 ** 24))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 8, 4), (3, 100, 37), (40, 64, 20)])
def test_the_lowest_planes_meet(tq, m, k, n):
    """x = 1 + 2^-8 + 255 2^-23 and f16 weights of 1 + 7 2^-10: the third plane of one and the second of the other are 2^-22.2 of
    the product, 3.4 half steps."""
    import torch

    v, w = 1 + 2.0 ** -8 + 255 * 2.0 ** -23, 1 + 7 * 2.0 ** -10
    x = torch.zeros(m, k, dtype=torch.float64, device="cuda")
    x[:, k - 1] = v
    for in_a in (True, False):
        a, b = torch.zeros(1, 1, k, device="cuda"), torch.zeros(1, n, 1, device="cuda")
        a[0, 0, k - 1], b[0, :, 0] = w if in_a else 1.0, 1.0 if in_a else w
        got = tq.Adapters(a.half(), b.half()).add(x.float(), torch.zeros(m, dtype=torch.int32, device="cuda"), torch.zeros(m, n, device="cuda"))
        assert float((got.double() / (v * w) - 1).abs().max()) <= 2.0 ** -23, in_a


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 20, 300, 1600])
@pytest.mark.parametrize("k,n", [(80, 40), (79, 1000)])
@pytest.mark.parametrize("dtype,weights", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float16"),
                                           ("float16", "bfloat16"), ("bfloat16", "float16")])
def test_rows_of_infinities_and_nan_are_not_finite(tq, m, k, n, dtype, weights):
    """Each output of a row that has one in x (its last element too) or in its adapter's a; the outputs of those in b."""
    import torch

    g = torch.Generator("cuda").manual_seed(m + k)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, y, index = f(m, k).to(getattr(torch, dtype)), f(m, n), torch.arange(m, dtype=torch.int32, device="cuda") % 6 - 1
    a, b = f(5, 1, 40, k).to(getattr(torch, weights)), f(5, n, 40).to(getattr(torch, weights))
    want = tq.Adapters(a, b).add(x, index, y)
    assert torch.isfinite(want).all()
    for bad in (float("nan"), float("inf"), -float("inf")):
        for column in (0, 3, k - 1):
            poisoned = x.clone()
            poisoned[1::7, column] = bad
            got = tq.Adapters(a, b).add(poisoned, index, y)
            rows = torch.zeros(m, dtype=torch.bool, device="cuda")
            rows[1::7] = True
            rows &= index >= 0
            assert not torch.isfinite(got[rows]).any() and torch.equal(got[~rows], want[~rows]), (bad, column)
            a2 = a.clone()
            a2[2, 0, 39, column] = bad
            got, rows = tq.Adapters(a2, b).add(x, index, y), index == 2
            assert not torch.isfinite(got[rows]).any() and torch.equal(got[~rows], want[~rows]), (bad, column)
        b2 = b.clone()
        b2[3, n - 1, 39], b2[0, 0, 0] = bad, bad
        got = tq.Adapters(a, b2).add(x, index, y)
        hit = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        hit[index == 3, n - 1], hit[index == 0, 0] = True, True
        assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit]), bad


def test_one_launch_is_for_rows_of_few_adapters():
    """A block takes the adapters that rows may name one after the other: a workspace says that they are two launches'."""
    from test_adapters import at, desc
    from theano_quantize import _abi

    need = lambda m, **kw: _abi.entry("tq_adapters_workspace_bytes")(at(desc(**dict(parts=1, rank=16, n=4096) | kw)), m)  # noqa: E731
    for m, count, k in ((1, 48, 4096), (16, 1, 256), (2, 2, 1024), (4, 4, 256), (16, 4, 256), (3, 3, 455)):
        assert need(m, count=count, k=k) == 0, (m, count, k)
    for m, count, k in ((1, 48, 4097), (16, 1, 257), (2, 2, 1025), (4, 4, 257), (5, 5, 16), (16, 16, 16), (16, 48, 256), (17, 1, 16)):
        assert need(m, count=count, k=k) > 0, (m, count, k)
