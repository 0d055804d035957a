"""Rotary positions of several axes (tq_rotary_apply_axes, tq_kv_write_rotary_axes): refusals on the CPU, numbers on the GPU."""
import ctypes

import pytest

from test_cache_abi import I64, batch, cache, heads, refuse, rotary, structure

TYPES = ("float32", "bfloat16", "float16")
Axes = structure(("axes", I64), ("position_stride", I64), ("planes0", ctypes.c_uint64), ("planes1", ctypes.c_uint64))


HELD = []


def at(x):
    """The address of a structure, which stays."""
    HELD.append(x)
    return None if x is None else ctypes.addressof(x)


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


def test_the_packed_descriptor_is_the_structure(abi):
    assert abi.rotary_axes_desc(3, 7, 1 << 63, 5) == bytes(Axes(3, 7, 1 << 63, 5))


@pytest.mark.parametrize("bad", [Axes(0, 3, 0, 0), Axes(5, 3, 0, 0), Axes(-1, 3, 0, 0), Axes(2, -3, 0, 0), Axes(2, 3, 2, 0),
                                 Axes(3, 3, 3 << 62, 0), Axes(1, 3, 1 << 40, 0), None])
def test_refusals(abi, bad):
    q, r, good = heads(abi), rotary(abi), Axes(2, 3, 1, 0)
    refuse(abi, "tq_rotary_apply_axes", at(r), at(bad), 256, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_kv_write_rotary_axes", at(cache(abi)), at(batch(abi)), at(r), at(bad), 256, at(q), at(q), at(q), 2, 256, None)
    refuse(abi, "tq_rotary_apply_axes", None, at(good), 256, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply_axes", at(r), at(good), None, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_kv_write_rotary_axes", at(cache(abi)), at(batch(abi)), at(r), at(good), 260, at(q), at(q), at(q), 2, 256, None)
    refuse(abi, "tq_kv_write_rotary_axes", at(cache(abi)), at(batch(abi)), None, at(good), 256, at(q), at(q), at(q), 2, 256, None)
    wide, big = rotary(abi, rotary_dim=4096), heads(abi, heads=0)  # more planes than the descriptor holds
    refuse(abi, "tq_rotary_apply_axes", at(wide), at(good), 256, 3, at(big), None, 2, 4096, 256, None, None)
    # planes past rotary_dim are nobody's
    abi.call("tq_rotary_apply_axes", at(rotary(abi, rotary_dim=62)), at(Axes(2, 3, 3 << 62, 7)), 256, 0, at(q), None, 2, 64, 256, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 200])
def test_heads_that_do_not_turn_read_no_axis(tq, n):
    """rotary_dim 0, whatever the words of the planes hold: the numbers as they are."""
    import torch
    from theano_quantize import _abi

    x, pos = torch.randn(n, 5, 64, device="cuda"), torch.arange(2 * n, device="cuda")
    out = torch.full_like(x, 7.0)
    _abi.call("tq_rotary_apply_axes", _abi.rotary_desc(0, 0, False, False, 1.0), _abi.rotary_axes_desc(2, n, 2 ** 64 - 1, 2 ** 64 - 1),
              pos.data_ptr(), n, _abi.heads_desc(x.data_ptr(), 5, x.stride(0), x.stride(1)), None, 2, 64, out.data_ptr(), None, None)
    torch.cuda.synchronize()
    assert torch.equal(out, x)


def axes_of(tq, order, half, count):
    if order == "turn":
        return tq.Rotary.axes_in_turn(half, count)
    return tq.Rotary.axes_in_blocks([half // count] * (count - 1) + [half - half // count * (count - 1)])


def turned_by_axes(x, pos, axes, f, m, pairs, inverse=False):
    """Each plane by itself, with tests/test_gpu_cache.py's exact angles and bound."""
    import torch
    from test_gpu_cache import turned

    r = 2 * len(axes)
    y, tol = x.double().cpu().clone(), torch.zeros(x.shape, dtype=torch.float64)
    for i, axis in enumerate(axes):
        both = [2 * i, 2 * i + 1] if pairs else [i, i + r // 2]
        part, bound = turned(x[..., both], pos[axis], f[i:i + 1], m, pairs, inverse)
        y[..., both], tol[..., both] = part, bound
    return y, tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,h,hk,d,r,pairs,order,count", [
    (1, 2, 1, 128, 128, False, "blocks", 3), (7, 3, 3, 80, 80, False, "turn", 3), (130, 4, 2, 64, 64, True, "blocks", 2),
    (5, 5, 1, 100, 50, True, "turn", 4), (200, 2, 2, 97, 56, False, "blocks", 4), (9, 1, 0, 128, 18, False, "turn", 2),
    (300, 1, 1, 128, 128, False, "turn", 4), (3, 1, 1, 2, 2, False, "blocks", 1), (129, 3, 1, 32, 8, True, "turn", 3)])
def test_numbers(tq, dtype, n, h, hk, d, r, pairs, order, count):
    import torch
    from test_gpu_cache import dtype_of, eps_half, least, rand

    dt = dtype_of(dtype)
    q, k = rand(n + d, n, h, d, dtype=dt), rand(n + d + 1, n, hk, d, dtype=dt) if hk else None
    axes = axes_of(tq, order, r // 2, count)
    rot = tq.Rotary.from_base(r, 10000.0, pairs, scale=1.25, axes=axes)
    pos = torch.randint(0, 1 << 20, (count, n), generator=torch.Generator().manual_seed(d)).cuda()
    for inverse in (False, True):
        for x, y in zip((q, k), rot.apply(q, k, pos, inverse=inverse)):
            if x is None:
                assert y is None
                continue
            ref, tol = turned_by_axes(x, pos, axes, rot.frequencies, 1.25, pairs, inverse)
            err = (y.double().cpu() - ref).abs()
            assert y.dtype == dt and y.shape == x.shape
            assert (err <= tol + eps_half(dt) * ref.abs() * (1 + 2.0 ** -20) + least(dt)).all(), float((err - tol).max())
            assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.gpu
@pytest.mark.parametrize("d,r,pairs,n", [(128, 128, False, 40), (97, 56, False, 200), (64, 64, True, 200), (100, 50, True, 3)])
def test_one_axis_strides_and_single_tokens_give_the_same_numbers(tq, d, r, pairs, n):
    import torch
    from test_gpu_cache import rand

    x = rand(d, n, 3, d)
    plain, rot = tq.Rotary.from_base(r, 1000.0, pairs), tq.Rotary.from_base(r, 1000.0, pairs, axes=axes_of(tq, "turn", r // 2, 3))
    same = torch.arange(n, device="cuda") * 37
    want = plain.apply(x, None, same)[0]
    assert torch.equal(rot.apply(x, None, same)[0], want)
    assert torch.equal(rot.apply(x, None, same.expand(3, n))[0], want)  # stride 0
    pos = torch.randint(0, 1 << 30, (5, 2 * n + 3), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    want = rot.apply(x, None, pos[:3, :n].contiguous())[0]
    assert torch.equal(rot.apply(x, None, pos[:, :n])[0], want)  # more rows than axes, rows apart
    for i in range(0, n, 19):
        assert torch.equal(rot.apply(x[i:i + 1], None, pos[:, i:i + 1])[0], want[i:i + 1])
    back = rot.apply(want, None, pos[:3, :n], inverse=True)[0]
    # there and back: 2 turns of at most 6 roundings of the plane's size
    size = x.abs().amax(-1, keepdim=True)
    assert ((back - x).abs() <= 2 * 6 * 2.0 ** -24 * 2 * 2 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", ["i8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,r,pairs,n", [(128, 128, False, 6), (80, 80, False, 150), (100, 48, True, 7), (64, 64, False, 130)])
def test_the_cache_stores_what_apply_gives(tq, codes, dtype, d, r, pairs, n):
    import torch
    from test_gpu_cache import Case, dtype_of, rand

    x, v = rand(d, n, 2, d, dtype=dtype_of(dtype)), rand(d + 1, n, 2, d, dtype=dtype_of(dtype))
    rot = tq.Rotary.from_base(r, 1000.0, pairs, axes=axes_of(tq, "blocks", r // 2, 3))
    pos = torch.randint(0, 5000, (3, n), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    a, b = (Case(tq, [n, 9], [n - 2, 2], 16, 2, d, codes) for _ in range(2))
    want = rot.apply(x.float(), None, pos)[0]
    assert torch.equal(a.cache.write_rotary(x, x, v, rot, a.batch, pos), want.to(x.dtype))
    b.cache.write(want, v.float(), b.batch)
    for name in ("k", "k_scale", "v", "v_scale"):
        assert torch.equal(getattr(a.cache, name), getattr(b.cache, name)), name
    # without positions every axis has the rows' places
    plain = tq.Rotary.from_base(r, 1000.0, pairs)
    assert torch.equal(a.cache.write_rotary(x, x, v, rot, a.batch), b.cache.write_rotary(x, x, v, plain, b.batch))
    assert torch.equal(a.cache.k, b.cache.k)


@pytest.mark.gpu
def test_what_python_refuses(tq):
    import torch

    f = torch.ones(4, dtype=torch.float64, device="cuda")
    for axes in ((0, 1, 2), (0, 1, 2, 4), (0, 1, 2, -1), (0, 0, 0, 0, 0)):
        with pytest.raises(tq.InvalidArgument):
            tq.Rotary(f, axes=axes)
    rot, q = tq.Rotary(f, axes=(0, 1, 2, 0)), torch.zeros(5, 1, 8, device="cuda")
    for pos in (torch.zeros(2, 5, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 5, dtype=torch.int32),
                torch.zeros(5, 3, dtype=torch.int64).t(), torch.zeros(6, dtype=torch.int64), torch.zeros(1, 3, 5, dtype=torch.int64)):
        with pytest.raises(tq.InvalidArgument):
            rot.apply(q, None, pos.cuda())
    with pytest.raises(tq.InvalidArgument):
        rot.apply(q, None, torch.zeros(3, 5, dtype=torch.int64))
    with pytest.raises(tq.InvalidArgument):
        tq.Rotary(f).apply(q, None, torch.zeros(1, 5, dtype=torch.int64, device="cuda"))  # no axes: positions are [tokens]
