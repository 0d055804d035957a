"""What the serving and block-scaled FP8 entry points refuse before a launch (CPU), and the largest that they take (GPU).
A launch holds less than 2^32 threads: 2^24 - 1 blocks of 256."""
import pytest

from test_cache_abi import abi, at, batch, cache, heads, rotary  # noqa: F401 (abi: a fixture)

BLOCKS = 1 << 24


def refuse(abi, name, *args):
    """`name` says that the call is past what a launch holds.  Structures are passed as they are (alive until the call)."""
    from theano_quantize import InvalidArgument

    with pytest.raises(InvalidArgument, match="blocks"):
        abi.call(name, *(at(x) if hasattr(x, "_fields_") else x for x in args))


def test_more_rows_than_a_launch_holds(abi):
    one, c = heads(abi, heads=1), cache(abi, heads=1)
    for n in (BLOCKS, 1 << 30):  # a block for each token
        refuse(abi, "tq_rotary_apply", rotary(abi), 256, n, one, None, 2, 64, 256, None, None)
    refuse(abi, "tq_rotary_apply", rotary(abi, rotary_dim=0), 256, 16 * BLOCKS - 15, one, None, 2, 64, 256, None, None)

    def of(rows):
        return batch(abi, batch=1, max_tokens=rows, tokens=rows)

    # 16 tokens to a block where heads are only coded, 4 where they turn or are read back
    refuse(abi, "tq_kv_write", c, of(16 * BLOCKS - 15), one, one, 2, None)
    refuse(abi, "tq_kv_write_rotary", c, of(4 * BLOCKS - 3), rotary(abi), None, one, one, one, 2, 256, None)
    refuse(abi, "tq_kv_read", c, of(4 * BLOCKS - 3), 2, 256, 256, None)


def test_more_heads_and_tiles_than_a_launch_holds(abi):
    c, q = cache(abi, heads=1), heads(abi, heads=1)
    many, most = (batch(abi, batch=n, tokens=n) for n in (BLOCKS, BLOCKS - 1))
    refuse(abi, "tq_kv_attention", c, many, q, 2, None, 0, 1.0, 256, 1 << 40, 256, None)
    ws = abi.entry("tq_kv_attention_workspace_bytes")
    assert ws(at(c), at(many), 1) == -1 and ws(at(c), at(most), 1) == 0


def test_fp8_blocks_past_a_launch(abi):
    refuse(abi, "tq_quantize_fp8_block", 256, 1 << 30, 1 << 10, 256, 256, None)
    refuse(abi, "tq_quantize_fp8_g128", 256, 2, 1 << 28, 128, 256, 256, None)
    for m, n, k in ((200, (1 << 31) - 200, 1 << 10), (300, (1 << 31) - 200, 1), (1 << 30, 300, 256)):
        refuse(abi, "tq_gemm_fp8_block", 256, 256, 256, 256, None, m, n, k, 256, 1 << 50, 256, None)
        if m < 1 << 30:  # (there the activations' coder refuses)
            assert abi.entry("tq_linear_fp8_block_workspace_bytes")(m, n, k) >= 0


def test_descriptors_whose_products_do_not_fit(abi):
    """2^60 pages of 16 tokens are 0 in 64 bits; sizes that every call refuses have no workspace."""
    from theano_quantize import InvalidArgument

    h = heads(abi)
    ws = abi.entry("tq_kv_attention_workspace_bytes")
    for c, b in ((cache(abi), batch(abi, table_pages=1 << 60, table_stride=1 << 60)),
                 (cache(abi, page=1 << 16), batch(abi, table_pages=1 << 48, table_stride=1 << 48))):
        for name, args in (("tq_kv_write", (at(h), at(h), 2, None)), ("tq_kv_read", (2, 256, 256, None)),
                           ("tq_kv_attention", (at(h), 2, None, 0, 1.0, 256, 1 << 40, 256, None))):
            with pytest.raises(InvalidArgument):
                abi.call(name, at(c), at(b), *args)
        assert ws(at(c), at(b), 2) == -1
    big = dict(table_pages=64, table_stride=64)
    for c, b in ((cache(abi), batch(abi, batch=1 << 31, tokens=1 << 31, **big)), (cache(abi), batch(abi, max_tokens=1 << 62, **big)),
                 (cache(abi, head_dim=1000), batch(abi, **big)), (cache(abi, page=1 << 20), batch(abi, **big)),
                 (cache(abi, head_dim=0), batch(abi, **big)), (cache(abi, page=24), batch(abi, **big))):
        assert ws(at(c), at(b), 2) == -1
    c, b = cache(abi), batch(abi, **big)
    assert ws(at(c), at(b), 2 << 20) == -1 and ws(at(c), at(b), 2) > 0


@pytest.mark.gpu
def test_weights_of_2_to_the_32_codes_back(tq):
    """16 GB of floats: the first rows, those about each 2^31st code and the last ones."""
    import torch

    n, k = (1 << 20) + 3, 1 << 12
    q = torch.randint(0, 127, (n, k), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    s = torch.rand((n + 127) // 128, k // 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    w = tq.dequantize_fp8_block(q, s)
    for r in (0, (1 << 19) - 100, (1 << 20) - 100, n - 100):
        part = slice(r, r + 100)
        grown = s[torch.arange(r, r + 100, device="cuda") // 128].repeat_interleave(128, 1)
        assert torch.equal(w[part], q[part].view(torch.float8_e4m3fn).float() * grown)


@pytest.mark.gpu
def test_rotary_of_as_many_tokens_as_a_launch_holds(tq):
    import torch

    n = BLOCKS - 1
    x = torch.randn(n, 1, 2, device="cuda", dtype=torch.float16, generator=torch.Generator("cuda").manual_seed(3))
    pos = torch.arange(n, device="cuda")
    rot = tq.Rotary.from_base(2)
    y = rot.apply(x, None, pos)[0]
    for i in (0, 1 << 23, n - 3):
        assert torch.equal(y[i:i + 3], rot.apply(x[i:i + 3], None, pos[i:i + 3])[0])


def test_fp8_block_layers_take_tensors_that_the_kernels_can_read():
    """Codes, scales and bias of one device, dense: the kernels take their addresses as they are."""
    import torch

    import theano_quantize as tq

    q, s, b = torch.zeros(300, 200, dtype=torch.uint8), torch.ones(3, 2), torch.zeros(300)
    assert tq.QuantizedLinear("fp8_block", 200, 300, q, s, b).bias is b
    for args in ((q, s.to("meta"), b), (q, s, b.to("meta")), (q.to("meta"), s, None), (q, s, torch.zeros(600)[::2]),
                 (q, s, torch.zeros(1).expand(300))):
        with pytest.raises(tq.InvalidArgument):
            tq.QuantizedLinear("fp8_block", 200, 300, *args)
