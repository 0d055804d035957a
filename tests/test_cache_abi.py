"""CPU checks of the serving entry points' refusals (rotary, cache, attention): every call below fails
validation, or has nothing to do, before anything is launched."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def abi():
    from theano_quantize import _abi

    return _abi


I64, PTR, I32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int32


def structure(*fields):
    """A descriptor of include/tq.h, laid out by ctypes apart from the package's own packing."""
    return type("Desc", (ctypes.Structure,), {"_fields_": list(fields)})


Heads = structure(("data", PTR), ("heads", I64), ("token_stride", I64), ("head_stride", I64))
RotaryDesc = structure(("frequencies", PTR), ("rotary_dim", I64), ("interleaved", I32), ("inverse", I32), ("scale", ctypes.c_float))
KVCacheDesc = structure(("k", PTR), ("k_scale", PTR), ("v", PTR), ("v_scale", PTR), ("pages", I64), ("heads", I64), ("page", I64),
                        ("head_dim", I64), ("codes", I32))
KVBatchDesc = structure(("table", PTR), ("table_stride", I64), ("table_pages", I64), ("lengths", PTR), ("offsets", PTR),
                        ("batch", I64), ("max_tokens", I64), ("tokens", I64))


def at(x):
    return None if x is None else ctypes.addressof(x)


def test_packed_descriptors_are_the_structures(abi):
    assert abi.heads_desc(1, 2, 3, 4) == bytes(Heads(1, 2, 3, 4))
    assert abi.rotary_desc(1, 2, 1, 0, 1.5) == bytes(RotaryDesc(1, 2, 1, 0, 1.5))
    assert abi.kv_cache_desc(1, 2, 3, 4, 5, 6, 7, 8, 3) == bytes(KVCacheDesc(1, 2, 3, 4, 5, 6, 7, 8, 3))
    assert abi.kv_batch_desc(1, 2, 3, 4, 5, 6, 7, 8) == bytes(KVBatchDesc(1, 2, 3, 4, 5, 6, 7, 8))


def cache(abi, **kw):
    d = dict(k=256, k_scale=256, v=256, v_scale=256, pages=4, heads=2, page=16, head_dim=64, codes=0)
    d.update(kw)
    return KVCacheDesc(**d)


def batch(abi, **kw):
    d = dict(table=256, table_stride=2, table_pages=2, lengths=256, offsets=None, batch=3, max_tokens=1, tokens=3)
    d.update(kw)
    return KVBatchDesc(**d)


def heads(abi, **kw):
    d = dict(data=256, heads=2, token_stride=128, head_stride=64)
    d.update(kw)
    return Heads(**d)


def rotary(abi, **kw):
    d = dict(frequencies=256, rotary_dim=64, interleaved=0, inverse=0, scale=1.0)
    d.update(kw)
    return RotaryDesc(**d)


def refuse(abi, name, *args):
    from theano_quantize import InvalidArgument

    with pytest.raises(InvalidArgument):
        abi.call(name, *args)
    assert abi.lib().tq_last_error().decode().startswith(name)


BAD_CACHE = [dict(codes=1), dict(codes=2), dict(head_dim=0), dict(head_dim=129), dict(page=8), dict(page=24), dict(page=0),
             dict(page=1 << 17), dict(heads=0), dict(heads=70000), dict(pages=0), dict(pages=1 << 31), dict(k=None),
             dict(v_scale=None), dict(k=264), dict(k_scale=260)]
BAD_BATCH = [dict(batch=-1), dict(tokens=-1), dict(max_tokens=-3), dict(table_pages=-1), dict(tokens=4), dict(lengths=None),
             dict(table=None), dict(lengths=258), dict(offsets=257, tokens=9), dict(table_stride=1),
             dict(table_pages=1 << 28, table_stride=1 << 28), dict(batch=1 << 31, tokens=1 << 31)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_caches(abi, kw):
    c, b, h = cache(abi, **kw), batch(abi), heads(abi)
    refuse(abi, "tq_kv_write", at(c), at(b), at(h), at(h), 2, None)
    refuse(abi, "tq_kv_read", at(c), at(b), 2, 256, 256, None)
    refuse(abi, "tq_kv_attention", at(c), at(b), at(h), 2, None, 0, 1.0, 256, 1 << 40, 256, None)
    r = rotary(abi, rotary_dim=0)
    refuse(abi, "tq_kv_write_rotary", at(c), at(b), at(r), None, at(h), at(h), at(h), 2, 256, None)


@pytest.mark.parametrize("kw", BAD_BATCH)
def test_bad_batches(abi, kw):
    c, b, h = cache(abi), batch(abi, **kw), heads(abi)
    refuse(abi, "tq_kv_write", at(c), at(b), at(h), at(h), 2, None)
    refuse(abi, "tq_kv_read", at(c), at(b), 2, 256, 256, None)
    refuse(abi, "tq_kv_attention", at(c), at(b), at(h), 2, None, 0, 1.0, 256, 1 << 40, 256, None)


def test_bad_rows(abi):
    c, b, h = cache(abi), batch(abi), heads(abi)
    for bad in (heads(abi, heads=3), heads(abi, data=None), heads(abi, data=257), heads(abi, token_stride=-1),
                heads(abi, head_stride=-64)):
        refuse(abi, "tq_kv_write", at(c), at(b), at(bad), at(h), 2, None)
        refuse(abi, "tq_kv_write", at(c), at(b), at(h), at(bad), 2, None)
        refuse(abi, "tq_kv_attention", at(c), at(b), at(bad), 2, None, 0, 1.0, 256, 1 << 40, 256, None)
    for dtype in (3, 7, -1):
        refuse(abi, "tq_kv_write", at(c), at(b), at(h), at(h), dtype, None)
        refuse(abi, "tq_kv_read", at(c), at(b), dtype, 256, 256, None)
        refuse(abi, "tq_kv_attention", at(c), at(b), at(h), dtype, None, 0, 1.0, 256, 1 << 40, 256, None)
    refuse(abi, "tq_kv_write", at(c), at(b), None, at(h), 2, None)
    refuse(abi, "tq_kv_write", None, at(b), at(h), at(h), 2, None)
    refuse(abi, "tq_kv_write", at(c), None, at(h), at(h), 2, None)
    refuse(abi, "tq_kv_read", at(c), at(b), 2, None, 256, None)
    refuse(abi, "tq_kv_read", at(c), at(b), 2, 256, 258, None)


def test_bad_rotary(abi):
    q = heads(abi)
    for kw in (dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=66), dict(frequencies=None)):
        r = rotary(abi, **kw)
        refuse(abi, "tq_rotary_apply", at(r), 256, 3, at(q), None, 2, 64, 256, None, None)
        refuse(abi, "tq_kv_write_rotary", at(cache(abi)), at(batch(abi)), at(r), None, at(q), at(q), at(q), 2, 256, None)
    r = rotary(abi)
    refuse(abi, "tq_rotary_apply", None, 256, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), None, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 260, 3, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 256, -1, at(q), None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 256, 3, at(q), None, 2, 64, None, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 256, 3, at(q), at(q), 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 256, 3, at(q), None, 9, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", at(r), 256, 3, at(q), None, 2, 130, 256, None, None)
    refuse(abi, "tq_kv_write_rotary", at(cache(abi)), at(batch(abi)), at(r), 12, at(q), at(q), at(q), 2, 256, None)
    refuse(abi, "tq_kv_write_rotary", at(cache(abi)), at(batch(abi)), at(r), None, at(q), at(q), at(q), 2, None, None)


def test_bad_attention(abi):
    c, b, h = cache(abi), batch(abi, table_pages=40, table_stride=40), heads(abi)
    need = abi.entry("tq_kv_attention_workspace_bytes")(at(c), at(b), 2)
    assert need > 0 and need % 4 == 0
    name = "tq_kv_attention"
    refuse(abi, name, at(c), at(b), at(h), 2, None, 0, 1.0, 256, need - 1, 256, None)   # workspace too small
    refuse(abi, name, at(c), at(b), at(h), 2, None, 0, 1.0, None, need, 256, None)
    refuse(abi, name, at(c), at(b), at(h), 2, None, 0, 1.0, 128, need, 256, None)       # not 256-byte aligned
    refuse(abi, name, at(c), at(b), at(h), 2, None, 0, 1.0, 256, need, None, None)      # no output
    refuse(abi, name, at(c), at(b), at(h), 2, None, 0, 1.0, 256, need, 258, None)
    refuse(abi, name, at(c), at(b), at(heads(abi, heads=3)), 2, None, 0, 1.0, 256, need, 256, None)
    refuse(abi, name, at(c), at(b), at(h), 2, 256, 0, 1.0, 256, need, 256, None)        # tree without words
    refuse(abi, name, at(c), at(b), at(h), 2, 258, 1, 1.0, 256, need, 256, None)
    many = batch(abi, max_tokens=33, tokens=99, table_pages=40, table_stride=40)
    refuse(abi, name, at(c), at(many), at(h), 2, 256, 1, 1.0, 256, 1 << 40, 256, None)  # 33 tokens, 32 bits
    huge = batch(abi, batch=1 << 20, tokens=1 << 20, table_pages=1 << 20, table_stride=1 << 20)
    refuse(abi, name, at(c), at(huge), at(h), 2, None, 0, 1.0, 256, 1 << 40, 256, None)  # 2^31 units of work
    ws = abi.entry("tq_kv_attention_workspace_bytes")
    assert ws(at(c), at(b), 3) == -1 and ws(None, at(b), 2) == -1 and ws(at(c), None, 2) == -1
    assert ws(at(c), at(batch(abi, batch=0, tokens=0)), 2) == 0
    assert ws(at(c), at(batch(abi)), 2) == 0  # 32 tokens: never split


def test_nothing_to_do(abi):
    c, h = cache(abi), heads(abi)
    for b in (batch(abi, batch=0, tokens=0), batch(abi, max_tokens=0, tokens=0)):
        assert abi.call("tq_kv_write", at(c), at(b), at(h), at(h), 2, None) == 0
        assert abi.call("tq_kv_read", at(c), at(b), 2, None, None, None) == 0
        assert abi.call("tq_kv_attention", at(c), at(b), at(h), 2, None, 0, 1.0, None, 0, None, None) == 0
    assert abi.call("tq_rotary_apply", at(rotary(abi)), None, 0, at(h), None, 2, 64, None, None, None) == 0


def test_python_refuses_host_tensors(abi):
    """The modules take device tensors of the stated types; what is wrong is said before any device work."""
    import torch

    import theano_quantize as tq

    with pytest.raises(tq.InvalidArgument):
        tq.Rotary(torch.ones(4, dtype=torch.float64))
    with pytest.raises(tq.InvalidArgument):
        tq.Rotary.from_base(7)
    with pytest.raises(tq.InvalidArgument):
        tq.Rotary.from_base(8, scaling="other")
    with pytest.raises(tq.InvalidArgument):
        tq.Rotary.from_base(8, scaling="yarn", factor=4.0)
    with pytest.raises(tq.InvalidArgument):
        tq.KVBatch(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    z = torch.zeros(2, 1, 16, 64, dtype=torch.int8)
    s = torch.zeros(2, 1, 16)
    for args in ((z, s, z, s, 64), (z.float(), s, z.float(), s, 64), (z, s, z, s, 65), (z, s[0], z, s, 64),
                 (z, s, z.to(torch.uint8), s, 64)):
        with pytest.raises(tq.InvalidArgument):
            tq.KVCache(*args)
    with pytest.raises(tq.InvalidArgument):
        tq.KVCache.allocate(2, 16, 1, 64, tq.QuantDType.Int4)
    with pytest.raises(tq.InvalidArgument):
        tq.tree_mask(torch.zeros(2, 2))


def test_tree_mask_words():
    import torch

    import theano_quantize as tq

    g = torch.Generator().manual_seed(3)
    for t in (1, 31, 32, 33, 64, 70):
        seen = torch.rand(5, t, generator=g) < 0.5
        w = tq.tree_mask(seen)
        assert w.dtype == torch.int32 and w.shape == (5, (t + 31) // 32)
        for i in range(5):
            for j in range(t):
                assert bool((int(w[i, j // 32]) >> (j % 32)) & 1) == bool(seen[i, j])
    assert tq.tree_mask(torch.zeros(0, 0, dtype=torch.bool)).shape == (0, 1)
