"""Performance cases of a decoder layer's serving operators on 8-bit state.

Four operators, as a program that serves a quantized decoder calls them: rotary positions on
the projections' output, the 8-bit key/value cache as it is written and read back, the
attention of new tokens over that cache, and the block-scaled FP8 projections around it.
With `own` set `run` makes the framework's calls; without, it computes the same in elementary
torch operations, so that both can be timed and compared on the same inputs.

Case fields by "kind":
  rope    n tokens, h query and hk key heads of width d, of which the first r columns turn,
          layout (half, pairs), scaling (none, linear, ntk, yarn), far: positions up to this, dtype
  cache   codes (i8, fp8), b sequences of about l tokens, the last t of each new, hk heads of width d,
          pages of `page` tokens; h > 0: h query heads and the keys turned on the way (rotary);
          read: new (the tokens written) or all; ragged; dtype in and `out` back
  attend  codes, b, l, t, h, hk, d, page, mask (causal, tree), ragged, dtype
  fp8     m tokens, n outputs, k inputs, bias
"""
import math
import os
import random
import sys

import torch

own = False

# ranges of the drawn cases (the listed ones lie inside them)
TOKENS = (1, 4096)            # tokens of a rotary, cache or Linear call
LENGTH = (1, 131072)          # cached tokens of a sequence
FAR = (64, 1 << 20)           # positions
WIDTH = (64, 16384)           # inputs and outputs of a layer
MAX_CACHE = 40 * 4096 * 8 * 128  # cached elements of keys (and of values)
MAX_PAIRS = 4.4e9             # query element times visible key: about the listed chunk's
MAX_FLOPS = 6.7e10            # of an FP8 product


def listed():
    return [
        # eight streams' next tokens in a grouped-head decoder, rotated in halves: the smallest call
        {"name": "rope_step", "kind": "rope", "n": 8, "h": 32, "hk": 8, "d": 128, "r": 128, "layout": "half",
         "scaling": "none", "far": 4096, "dtype": "f32"},
        # an odd-length prompt at the far end of a stretched context, half of each head turned in pairs
        {"name": "rope_far_prompt", "kind": "rope", "n": 4093, "h": 32, "hk": 32, "d": 128, "r": 64, "layout": "pairs",
         "scaling": "yarn", "far": 1 << 20, "dtype": "bf16"},
        # one decoding step of sixteen streams: rotate q, rotate and store k, store v, look at what was stored
        {"name": "cache_step", "kind": "cache", "codes": "i8", "b": 16, "l": 1000, "t": 1, "h": 32, "hk": 8, "d": 128,
         "page": 64, "read": "new", "ragged": True, "dtype": "bf16", "out": "bf16"},
        # a prompt of a model with 80-wide heads stored as FP8 and read back for the layer's own f32 attention
        {"name": "cache_prompt", "kind": "cache", "codes": "fp8", "b": 2, "l": 2048, "t": 2048, "h": 0, "hk": 32, "d": 80,
         "page": 16, "read": "new", "ragged": False, "dtype": "f32", "out": "f32"},
        # a token joins a long context, which is read back whole (moved off the card, or to another form)
        {"name": "cache_read_long", "kind": "cache", "codes": "i8", "b": 1, "l": 32767, "t": 1, "h": 0, "hk": 8, "d": 128,
         "page": 64, "read": "all", "ragged": False, "dtype": "f32", "out": "f32"},
        # one stream's next token over a short context: latency
        {"name": "attend_step", "kind": "attend", "codes": "i8", "b": 1, "l": 777, "t": 1, "h": 32, "hk": 8, "d": 128,
         "page": 64, "mask": "causal", "ragged": False, "dtype": "bf16"},
        # a full serving batch of ragged contexts
        {"name": "attend_batch", "kind": "attend", "codes": "i8", "b": 64, "l": 4096, "t": 1, "h": 32, "hk": 8, "d": 128,
         "page": 64, "mask": "causal", "ragged": True, "dtype": "f32"},
        # one stream at the far end of a long context, FP8 cache
        {"name": "attend_long", "kind": "attend", "codes": "fp8", "b": 1, "l": 131071, "t": 1, "h": 32, "hk": 8, "d": 128,
         "page": 256, "mask": "causal", "ragged": False, "dtype": "bf16"},
        # trees of drafted tokens to be verified, eight streams, heads of 64 without grouping
        {"name": "attend_tree", "kind": "attend", "codes": "i8", "b": 8, "l": 2048, "t": 48, "h": 16, "hk": 16, "d": 64,
         "page": 32, "mask": "tree", "ragged": True, "dtype": "f32"},
        # a chunk of a prompt behind what is cached of it
        {"name": "attend_chunk", "kind": "attend", "codes": "fp8", "b": 1, "l": 2500, "t": 500, "h": 32, "hk": 8, "d": 128,
         "page": 64, "mask": "causal", "ragged": False, "dtype": "bf16"},
        # a token through the widest projection of a 4096-wide model
        {"name": "fp8_decode", "kind": "fp8", "m": 1, "n": 14336, "k": 4096, "bias": False},
        # a prompt through the square projection, a length and width off every tile
        {"name": "fp8_prompt", "kind": "fp8", "m": 2047, "n": 4104, "k": 4000, "bias": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["rope", "cache", "attend", "fp8"], [15, 20, 40, 25])[0]
    dtype = rng.choice(["f32", "bf16", "f16"])
    d = rng.choice([32, 40, 64, 64, 72, 80, 96, 100, 128, 128, 128])
    hk = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    h = hk * rng.choice([1, 1, 2, 4, 4, 7, 8])
    if kind == "rope":
        n = min(_log(rng, *TOKENS), max(1, 4093 * 64 // (h + hk)))
        return {"kind": kind, "n": n, "h": h, "hk": hk, "d": d, "r": rng.choice([d, d, 2 * rng.randint(1, d // 2)]),
                "layout": rng.choice(["half", "pairs"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
                "far": _log(rng, *FAR), "dtype": dtype}
    page, codes = rng.choice([16, 32, 48, 64, 128, 256]), rng.choice(["i8", "fp8"])
    b, ragged = _log(rng, 1, 64), rng.random() < 0.6
    if kind == "cache":
        t = rng.choice([1, 1, _log(rng, 1, 64), _log(rng, *TOKENS)])
        l = max(t, _log(rng, 1, 32768))
        read = rng.choice(["new", "new", "all"])
        while b * l * hk * d > MAX_CACHE // 8 or b * t * (h + hk) * d > 4096 * 64 * 128:
            if b > 1:
                b = (b + 1) // 2
            else:
                l = (l + 1) // 2
                t = min(t, l)
        h = rng.choice([0, h])  # turned keys lie anywhere between two codes: their values are read in 16 bits
        out = dtype if dtype != "f32" else rng.choice(["bf16", "f16"] if h else ["f32", "bf16", "f16"])
        return {"kind": kind, "codes": codes, "b": b, "l": l, "t": t, "h": h, "hk": hk, "d": d, "page": page,
                "read": read, "ragged": ragged, "dtype": dtype, "out": out}
    if kind == "attend":
        t = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 2, 128), _log(rng, 64, 600)])
        l = max(t, _log(rng, *LENGTH))
        while b * l * hk * d > MAX_CACHE or b * t * h * d * l > MAX_PAIRS:
            if b > 1:
                b = (b + 1) // 2
            elif l > t:
                l = max(t, (l + 1) // 2)
            else:
                t = l = (t + 1) // 2
        return {"kind": kind, "codes": codes, "b": b, "l": l, "t": t, "h": h, "hk": hk, "d": d, "page": page,
                "mask": rng.choice(["causal", "tree"]) if t <= 128 else "causal", "ragged": ragged, "dtype": dtype}
    n, k = (128 * _log(rng, 1, 128) if rng.random() < 0.5 else _log(rng, *WIDTH) for _ in range(2))
    while n * k > 14336 * 8192:
        n = (n + 1) // 2
    return {"kind": kind, "m": min(_log(rng, *TOKENS), max(1, int(MAX_FLOPS / (2 * n * k)))), "n": n, "k": k,
            "bias": rng.random() < 0.5}


# ------------------------------------------------------------------ geometry
def _lengths(case):
    """Cached tokens of each sequence, the new ones among them: ragged batches go down to a quarter."""
    b, l, t = case["b"], case["l"], case["t"]
    return [max(t, l - (l * 3 // 4) * (i * 61 % 97) // 97) if case["ragged"] else l for i in range(b)]


def _new(case):
    """New tokens of each sequence: those of a ragged batch differ (where there are several)."""
    t = case["t"]
    return [max(1, t - (i * 37 % 11) * t // 16) if case["ragged"] else t for i in range(case["b"])]


def _padded(d):
    return (d + 31) // 32 * 32


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_YARN = {"factor": 32.0, "original": 32768, "fast": 32.0, "slow": 1.0}


def _frequencies(case):
    """Angles per position (f64, on the host) of a rotary case, and the factor of its outputs."""
    r = case["r"] if case["kind"] == "rope" else case["d"] // 2 * 2
    scaling = case.get("scaling", "none")
    base = 10000.0 if scaling != "ntk" else 10000.0 * 8.0 ** (r / max(1.0, r - 2.0))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if scaling == "linear":
        return f / 8.0, 1.0
    if scaling != "yarn":
        return f, 1.0
    y = _YARN
    edge = [r * math.log(y["original"] / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (y["fast"], y["slow"])]
    lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
    ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return f / y["factor"] * ramp + f * (1.0 - ramp), 0.1 * math.log(y["factor"]) + 1.0


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _normal(g, shape, std=1.0, dtype="f32"):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(_TYPES[dtype])


def _stored(g, case, pages):
    """Codes and scales of a cache in use: tokens of differing size, and stale ones where no token lies."""
    rows, d = pages * case["hk"] * case["page"], case["d"]
    x = _normal(g, (rows, d))
    x *= torch.rand(rows, 1, generator=g, device="cuda") + 0.5
    top = 127.0 if case["codes"] == "i8" else 448.0
    s = (x.abs().amax(1) / top).clamp_min(1e-10)
    x /= s[:, None]
    c = x.round_().to(torch.int8) if case["codes"] == "i8" else x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    full = torch.zeros(rows, _padded(d), dtype=c.dtype, device="cuda")
    full[:, :d] = c
    shape = (pages, case["hk"], case["page"])
    return full.view(*shape, -1), s.view(shape)


def _tree(rng, counts):
    """Bit words [tokens, words] of trees of drafted tokens: each sees itself and its ancestors."""
    words, rows = (max(counts) + 31) // 32, []
    for n in counts:
        seen = []
        for t in range(n):
            up = rng.randint(max(-1, t - 5), t - 1)
            seen.append((seen[up] if up >= 0 else 0) | 1 << t)
        rows += [[((v >> 32 * w) & 0xFFFFFFFF) for w in range(words)] for v in seen]
    full = torch.tensor(rows, dtype=torch.int64)
    return torch.where(full >= 1 << 31, full - (1 << 32), full).to(torch.int32).cuda()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "rope":
        f, m = _frequencies(case)
        n, d, far = case["n"], case["d"], case["far"]
        pos = torch.randint(far // 2, far, (n,), generator=g, device="cuda") if n < 64 else \
            torch.arange(n, device="cuda") + (far - n if far > n else 0)
        if n >= 64:
            pos = pos + torch.randint(0, 3, (1,), generator=g, device="cuda")
        return {"case": case, "q": _normal(g, (n, case["h"], d), 1.0, case["dtype"]),
                "k": _normal(g, (n, case["hk"], d), 1.0, case["dtype"]), "positions": pos, "frequencies": f.cuda(), "m": m}
    if kind == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        w = _normal(g, (n, k), 0.02)
        nb, kb = (n + 127) // 128, (k + 127) // 128
        full = torch.zeros(nb * 128, kb * 128, device="cuda")
        full[:n, :k] = w
        s = (full.view(nb, 128, kb, 128).abs().amax((1, 3)) / 448.0).clamp_min(1e-10)
        grown = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        codes = (w / grown).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return {"case": case, "x": _normal(g, (m, k)), "codes": codes, "scales": s,
                "bias": _normal(g, (n,), 0.1) if case["bias"] else None}
    lengths, new = _lengths(case), _new(case)
    per = max((v + case["page"] - 1) // case["page"] for v in lengths)
    pages = case["b"] * per + 3
    table = torch.randperm(pages, generator=g, device="cuda")[:case["b"] * per].view(case["b"], per).to(torch.int32)
    (kc, ks), (vc, vs) = _stored(g, case, pages), _stored(g, case, pages)
    offsets = [sum(new[:i]) for i in range(case["b"] + 1)]
    n, d = offsets[-1], case["d"]
    s = {"case": case, "k_cache": kc, "k_scale": ks, "v_cache": vc, "v_scale": vs, "table": table, "n": n,
         "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(), "offsets": torch.tensor(offsets, dtype=torch.int32).cuda(),
         "all_offsets": torch.tensor([sum(lengths[:i]) for i in range(case["b"] + 1)], dtype=torch.int32).cuda(),
         "n_all": sum(lengths), "longest": max(lengths), "most": max(new)}
    if kind == "cache":
        s["k"] = _normal(g, (n, case["hk"], d), 1.0, case["dtype"])
        s["v"] = _normal(g, (n, case["hk"], d), 0.7, case["dtype"])
        if case["h"]:
            f, s["m"] = _frequencies(case)
            s["q"], s["frequencies"] = _normal(g, (n, case["h"], d), 1.0, case["dtype"]), f.cuda()
        return s
    s["q"] = _normal(g, (n, case["h"], d), 1.5, case["dtype"])
    s["tree"] = _tree(random.Random(int(seed) * 7 + 3), new) if case["mask"] == "tree" else None
    return s


# ------------------------------------------------------------------ the plain forms
def _turn(x, positions, f, m, layout):
    a = positions.double()[:, None] * f  # far positions lose their angle in 32 bits
    c, s = (a.cos() * m).float()[:, None], (a.sin() * m).float()[:, None]
    r, v = 2 * f.numel(), x.float()
    if layout == "half":
        p, q = v[..., :r // 2], v[..., r // 2:r]
        turned = torch.cat([p * c - q * s, q * c + p * s], -1)
    else:
        p, q = v[..., 0:r:2], v[..., 1:r:2]
        turned = torch.stack([p * c - q * s, q * c + p * s], -1).flatten(-2)
    return torch.cat([turned, v[..., r:]], -1)


def _coded(x, kind):
    """Codes and scales of each token's heads: quotients in 64 bits for INT8, whose ties round away from zero."""
    s = (x.abs().amax(-1).double() / (127.0 if kind == "i8" else 448.0)).clamp_min(1e-10).float()
    if kind == "i8":
        v = x.double() / s.double()[..., None]
        return (v.abs() + 0.5).floor().copysign(v).clamp(-128, 127).to(torch.int8), s
    return (x / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s


def _floats(codes):
    return codes.float() if codes.dtype == torch.int8 else codes.view(torch.float8_e4m3fn).float()


def _places(s, offsets, n):
    """The sequence of each of n token rows, and its position there."""
    row = torch.arange(n, device="cuda")
    b = torch.searchsorted(offsets[1:].long(), row, right=True)
    return b, row - offsets[b + 1] + s["lengths"][b]


def _gathered(cache, scale, pages, off, d):
    return _floats(cache[pages, :, off, :d]) * scale[pages, :, off][..., None]


def _plain_cache(s):
    case, page = s["case"], s["case"]["page"]
    b, pos = _places(s, s["offsets"], s["n"])
    pages, off = s["table"][b, pos // page].long(), pos % page
    k, v, out = s["k"].float(), s["v"].float(), []
    if case["h"]:
        out.append(_turn(s["q"], pos, s["frequencies"], s["m"], "half").to(s["q"].dtype))
        k = _turn(s["k"], pos, s["frequencies"], s["m"], "half")
    for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        c, sc = _coded(x, case["codes"])
        cache[pages, :, off, :case["d"]] = c
        scale[pages, :, off] = sc
    if case["read"] == "all":
        b, pos = _places(s, s["all_offsets"], s["n_all"])
        pages, off = s["table"][b, pos // page].long(), pos % page
    kind = _TYPES[case["out"]]
    return out + [_gathered(s["k_cache"], s["k_scale"], pages, off, case["d"]).to(kind),
                  _gathered(s["v_cache"], s["v_scale"], pages, off, case["d"]).to(kind)]


def _whole(cache, scale, table, length, d):
    """[batch, heads, length, d] floats of every sequence's pages."""
    b, p = table.shape
    x = _floats(cache[table.long()][..., :d]) * scale[table.long()][..., None]  # [b, p, heads, page, d]
    return x.transpose(1, 2).reshape(b, cache.shape[1], -1, d)[:, :, :length]


def _plain_attend(s):
    case = s["case"]
    d, h, hk, most, length = case["d"], case["h"], case["hk"], s["most"], s["longest"]
    k = _whole(s["k_cache"], s["k_scale"], s["table"], length, d)
    v = _whole(s["v_cache"], s["v_scale"], s["table"], length, d)
    b, t = s["table"].shape[0], torch.arange(most, device="cuda")
    first, count = s["offsets"][:-1].long(), (s["offsets"][1:] - s["offsets"][:-1]).long()
    rows = (first[:, None] + t).clamp_max(s["n"] - 1)  # rows past a sequence's own are left out below
    q = s["q"].float()[rows].view(b, most, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    key, start = torch.arange(length, device="cuda"), (s["lengths"].long() - count)[:, None, None]
    draft = key[None, None] - start  # each key's place among the new tokens, negative before them
    if s["tree"] is None:
        seen = draft <= t[None, :, None]
    else:
        j = draft.clamp(0, 32 * s["tree"].shape[1] - 1)
        word = s["tree"][rows].long().gather(2, (j >> 5).expand(b, most, length))
        seen = (draft < 0) | ((draft < count[:, None, None]) & ((word >> (j & 31)) & 1 == 1))
    seen = seen & (key[None, None] < s["lengths"][:, None, None])
    scores = scores.view(b, hk, h // hk, most, length).masked_fill(~seen[:, None, None], float("-inf"))
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    o = torch.matmul(p.view(b, hk, -1, length), v).view(b, h, most, d) / p.sum(-1).view(b, h, most, 1)
    at, _ = _places(s, s["offsets"], s["n"])
    return o.transpose(1, 2)[at, torch.arange(s["n"], device="cuda") - first[at]].to(s["q"].dtype)


def _plain_fp8(s):
    x, (m, k) = s["x"], s["x"].shape
    kb = s["scales"].shape[1]
    full = torch.zeros(m, kb * 128, device="cuda")
    full[:, :k] = x
    full = full.view(m, kb, 128)
    sa = (full.abs().amax(-1).double() / 448.0).clamp_min(1e-10).float()
    a = (full / sa[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).float() * sa[..., None]
    n = s["codes"].shape[0]
    w = _floats(s["codes"]) * s["scales"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = a.view(m, -1)[:, :k] @ w.t()
    return y if s["bias"] is None else y + s["bias"]


# ------------------------------------------------------------------ the framework's calls
def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neo-theano_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import theano_quantize

    return theano_quantize


def _own_run(s):
    tq, case = _framework(), s["case"]
    if case["kind"] == "rope":
        return tq.Rotary(s["frequencies"], case["layout"] == "pairs", s["m"]).apply(s["q"], s["k"], s["positions"])
    if case["kind"] == "fp8":
        n, k = s["codes"].shape
        return tq.QuantizedLinear("fp8_block", k, n, s["codes"], s["scales"], s["bias"])(s["x"])
    cache = tq.KVCache(s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], case["d"])
    if case["ragged"]:
        new = tq.KVBatch(s["table"], s["lengths"], s["most"], s["offsets"], s["n"])
    else:
        new = tq.KVBatch(s["table"], s["lengths"], case["t"])
    if case["kind"] == "attend":
        return cache.attention(s["q"], new, tree=s["tree"])
    if case["h"]:
        out = [cache.write_rotary(s["q"], s["k"], s["v"], tq.Rotary(s["frequencies"], False, s["m"]), new)]
    else:
        cache.write(s["k"], s["v"], new)
        out = []
    if case["read"] == "all":
        new = tq.KVBatch(s["table"], s["lengths"], s["longest"], s["all_offsets"], s["n_all"])
    return out + list(cache.read(new, _TYPES[case["out"]]))


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["kind"] == "rope":
        return tuple(_turn(x, state["positions"], state["frequencies"], state["m"], case["layout"]).to(x.dtype)
                     for x in (state["q"], state["k"]))
    return {"fp8": _plain_fp8, "cache": _plain_cache, "attend": _plain_attend}[case["kind"]](state)


# ------------------------------------------------------------------ the definition in 64 bits
def _rotate64(x, positions, case):
    """Complex numbers times e^(i angle)."""
    f, m = _frequencies(case)
    r, x = 2 * f.numel(), x.double()
    turn = torch.polar(torch.full_like(f, m).cuda().expand(x.shape[0], -1).contiguous(),
                       positions.double()[:, None] * f.cuda())[:, None]
    if case.get("layout", "half") == "half":
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., r:]], -1)
    z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1)


def _e4m3(codes):
    """Values of e4m3 bit patterns in 64 bits."""
    c = codes.long()
    e, f = c >> 3 & 15, (c & 7).double()
    size = torch.where(e > 0, (1 + f / 8) * torch.exp2(e.double() - 7), f * 2.0 ** -9)
    return torch.where(c > 127, -size, size)


def _to_e4m3(x):
    """The e4m3 value nearest to x (|x| <= 448, ties to even), in 64 bits."""
    e = torch.frexp(x.abs().clamp_min(2.0 ** -6))[1].double() - 1  # normals from 2^-6 up; one step below
    step = torch.exp2(e - 3)
    return (x / step).round() * step


def _value64(x, kind):
    """What a token's head is stored as: scale and quotient are 32-bit numbers by definition (the INT8 quotient is not)."""
    s = (x.abs().amax(-1, keepdim=True) / (127.0 if kind == "i8" else 448.0)).clamp_min(1e-10).float().double()
    if kind == "i8":
        v = x / s
        return torch.sign(v) * (v.abs() + 0.5).floor() * s
    return _to_e4m3((x / s).float().double().clamp(-448, 448)) * s


def _dense64(cache, scale, table, length, d):
    """One sequence's [heads, length, d] in 64 bits."""
    page = cache.shape[2]
    pages = table[:(length + page - 1) // page].long()
    c = cache[pages][..., :d]
    x = (_e4m3(c) if c.dtype == torch.uint8 else c.double()) * scale[pages].double()[..., None]
    return x.permute(1, 0, 2, 3).reshape(cache.shape[1], -1, d)[:, :length].contiguous()


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        return tuple(_rotate64(s[x], s["positions"], case) for x in ("q", "k"))
    if kind == "fp8":
        x, k = s["x"].double(), case["k"]
        y = 0
        for i in range(0, k, 128):
            a = _value64(x[:, i:i + 128], "fp8")
            w = _e4m3(s["codes"][:, i:i + 128]) * s["scales"][:, i // 128].double().repeat_interleave(128)[:case["n"], None]
            y = y + a @ w.t().contiguous()
        return y if s["bias"] is None else y + s["bias"].double()
    d, lengths, new = case["d"], _lengths(case), _new(case)
    starts = [sum(new[:i]) for i in range(len(new))]
    if kind == "cache":
        pos = torch.cat([torch.arange(n - t, n) for n, t in zip(lengths, new)]).cuda()
        k, v = s["k"].double(), s["v"].double()
        out = []
        if case["h"]:
            k = _rotate64(k, pos, case)
            out.append(_rotate64(s["q"], pos, case))
        for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
            x = _value64(x, case["codes"])
            if case["read"] == "all":
                parts = []
                for i, (n, t) in enumerate(zip(lengths, new)):
                    old = _dense64(cache, scale, s["table"][i], n, d).transpose(0, 1)[:n - t]
                    parts += [old, x[starts[i]:starts[i] + t]]
                x = torch.cat(parts)
            out.append(x)
        return out
    out = []
    for i, (n, t) in enumerate(zip(lengths, new)):
        k = _dense64(s["k_cache"], s["k_scale"], s["table"][i], n, d)
        v = _dense64(s["v_cache"], s["v_scale"], s["table"][i], n, d)
        q = s["q"][starts[i]:starts[i] + t].double().transpose(0, 1).reshape(case["hk"], -1, d)
        score = (q @ k.transpose(1, 2).contiguous() / math.sqrt(d)).view(case["h"], t, n)
        if s["tree"] is None:
            hidden = torch.ones(t, t, device="cuda").triu(1).bool()
        else:
            words = s["tree"][starts[i]:starts[i] + t].cpu().tolist()
            hidden = torch.tensor([[not (words[a][j // 32] >> (j % 32)) & 1 for j in range(t)] for a in range(t)]).cuda()
        score[..., n - t:].masked_fill_(hidden, float("-inf"))
        o = torch.softmax(score, -1).view(case["hk"], -1, n) @ v
        out.append(o.view(case["h"], t, d).transpose(0, 1))
    return torch.cat(out)


# ------------------------------------------------------------------ the work
def work(case):
    kind = case["kind"]
    if kind == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + 4 * ((n + 127) // 128) * ((k + 127) // 128) + 4 * m * (n + k) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    size = _SIZE[case["dtype"]]
    if kind == "rope":
        n, heads = case["n"], case["h"] + case["hk"]
        return {"bytes": 2 * n * heads * case["d"] * size + 8 * n + 4 * case["r"], "flops": 3 * n * heads * case["r"]}
    n, row = sum(_new(case)), case["hk"] * (case["d"] + 4) * 2  # a token's keys and values: codes and scales
    if kind == "cache":
        back = sum(_lengths(case)) if case["read"] == "all" else n
        moved = n * case["d"] * size * 2 * (case["hk"] + case["h"]) + n * row  # written
        moved += back * (row + 2 * case["hk"] * case["d"] * _SIZE[case["out"]])  # and read back
        return {"bytes": moved, "flops": 3 * n * case["d"] * (case["h"] + case["hk"])}
    pairs = sum(t * (l - t) + t * (t + 1) // 2 for l, t in zip(_lengths(case), _new(case)))
    return {"bytes": sum(_lengths(case)) * row + 2 * n * case["h"] * case["d"] * size, "flops": 4 * pairs * case["h"] * case["d"]}
