"""Performance cases of what serving many requests adds to a quantized decoder layer.

Four operators, as a program that serves drafted tokens for many requests calls them: low-rank
adapters of each request beside a shared projection, rotary positions with several axes (time,
height, width), the verification of drafted tokens against the target's probabilities, and the
cache's pages as sequences fork, grow, end and keep what was verified.  With `own` set `run`
makes the framework's calls; without, it computes the same in elementary torch operations, so
that both can be timed and compared on the same inputs.

Case fields by "kind":
  adapt   m tokens, count adapters of rank r, k inputs, n outputs in `parts` slices with adapters of
          their own (a fused projection), rows: mixed (a request a row) or runs (a prompt a run),
          dtype of x, weights of a and b
  turn    n tokens, h query and hk key heads of width d, of which r columns turn, `axes` axes whose
          planes lie in blocks or in turn, layout (half, pairs), dtype; store: k and v go to a cache
          (codes, page) and come back in `out`
  verify  b sequences of t new tokens (ragged: fewer), vocab, tree (up to `width` children to a token)
          or chain, draft: the draft model's probabilities are there, dtype of the probabilities
  pages   do: keep (the verified path of t new tokens of b sequences) or fork (b sequences into n
          children, which grow by t tokens, and end), about l tokens in each, pages of `page` tokens,
          hk heads of width d, codes
"""
import math
import os
import random
import sys

import torch

own = False

# ranges of the drawn cases (the listed ones lie inside them)
TOKENS = (1, 4096)      # tokens of an adapter or rotary call
WIDTH = (64, 16384)     # inputs and outputs of a layer
VOCAB = (1000, 262144)  # tokens that a model knows
MAX_MOVED = 5e8        # bytes of an adapter call's rows
MAX_ADAPTERS = 1.2e8    # bytes of a call's adapters
MAX_PROBS = 3.3e7       # probabilities of a verification (of each model)
MAX_CACHE = 6e7         # bytes of a cache's keys (and of its values)


def listed():
    return [
        # one request's next token through a square projection: the smallest call
        {"name": "adapt_token", "kind": "adapt", "m": 1, "count": 4, "r": 16, "parts": 1, "k": 4096, "n": 4096, "rows": "mixed",
         "dtype": "bf16", "weights": "bf16"},
        # a full serving batch, nearly every request with an adapter of its own, the widest projection
        {"name": "adapt_batch", "kind": "adapt", "m": 64, "count": 48, "r": 16, "parts": 1, "k": 4096, "n": 14336, "rows": "mixed",
         "dtype": "f32", "weights": "bf16"},
        # drafted tokens of a few requests through fused query, key and value projections
        {"name": "adapt_fused", "kind": "adapt", "m": 47, "count": 8, "r": 64, "parts": 3, "k": 2048, "n": 6144, "rows": "runs",
         "dtype": "f16", "weights": "f16"},
        # prompts of several requests in one call, some without an adapter
        {"name": "adapt_prompt", "kind": "adapt", "m": 4093, "count": 6, "r": 64, "parts": 1, "k": 4096, "n": 14336, "rows": "runs",
         "dtype": "f32", "weights": "bf16"},
        # eight streams' next tokens after images: positions of three axes, keys and values stored
        {"name": "turn_step", "kind": "turn", "n": 8, "h": 32, "hk": 8, "d": 128, "r": 128, "axes": 3, "order": "blocks",
         "layout": "half", "dtype": "bf16", "store": True, "codes": "i8", "page": 64, "out": "bf16"},
        # a large image's patches, planes of the axes in turn, heads of 80
        {"name": "turn_image", "kind": "turn", "n": 4087, "h": 16, "hk": 16, "d": 80, "r": 80, "axes": 3, "order": "turn",
         "layout": "half", "dtype": "f32", "store": False},
        # one stream's chain of drafted tokens, a small vocabulary: latency
        {"name": "verify_chain", "kind": "verify", "b": 1, "t": 6, "vocab": 32000, "tree": False, "draft": True, "width": 1,
         "dtype": "f32", "ragged": False},
        # a batch of chains over a large vocabulary
        {"name": "verify_batch", "kind": "verify", "b": 32, "t": 8, "vocab": 128256, "tree": False, "draft": True, "width": 1,
         "dtype": "f32", "ragged": True},
        # trees of a draft model's likeliest tokens, no probabilities of its own
        {"name": "verify_tree", "kind": "verify", "b": 8, "t": 48, "vocab": 32001, "tree": True, "draft": False, "width": 4,
         "dtype": "bf16", "ragged": True},
        # trees of tokens that were drawn from the draft model's probabilities
        {"name": "verify_drawn", "kind": "verify", "b": 4, "t": 24, "vocab": 128256, "tree": True, "draft": True, "width": 3,
         "dtype": "f32", "ragged": False},
        # the verified paths of those trees stay in the cache, the other branches go
        {"name": "keep_trees", "kind": "pages", "do": "keep", "codes": "i8", "b": 8, "l": 2048, "t": 48, "hk": 16, "d": 64,
         "page": 32, "n": 0},
        # sixteen prompts become four samples each: whole pages are shared, the begun ones copied
        {"name": "fork_samples", "kind": "pages", "do": "fork", "codes": "fp8", "b": 16, "l": 2000, "t": 4, "hk": 8, "d": 128,
         "page": 64, "n": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["adapt", "turn", "verify", "pages"], [40, 15, 25, 20])[0]
    dtype = rng.choice(["f32", "bf16", "f16"])
    d = rng.choice([32, 40, 64, 64, 72, 80, 96, 100, 128, 128, 128])
    hk = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    codes, page = rng.choice(["i8", "fp8"]), rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "adapt":
        m, parts, count = rng.choice([_log(rng, 1, 64), _log(rng, *TOKENS)]), rng.choice([1, 1, 1, 2, 3]), _log(rng, 1, 64)
        k, n = (128 * _log(rng, 1, 128) if rng.random() < 0.6 else _log(rng, *WIDTH) for _ in range(2))
        r = rng.choice([4, 8, 8, 16, 16, 32, 64, 12, 128])
        n = max(1, min(n, 16384) // parts) * parts
        while count > 1 and count * r * (parts * k + n) * 2 > MAX_ADAPTERS:
            count = (count + 1) // 2
        m = min(m, max(1, int(MAX_MOVED / (4 * k + 8 * n))))
        if m > 64:
            count = min(count, 12)
        return {"kind": kind, "m": m, "count": count, "r": r, "parts": parts, "k": k, "n": n,
                "rows": rng.choice(["mixed", "runs"]) if m <= 64 else "runs", "dtype": dtype, "weights": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "turn":
        h, store = hk * rng.choice([1, 1, 2, 4, 4, 7, 8]), rng.random() < 0.5
        n = min(_log(rng, *TOKENS), max(1, 4096 * 40 // (h + hk)))
        case = {"kind": kind, "n": n, "h": h, "hk": hk, "d": d, "r": rng.choice([d, d, 2 * rng.randint(4, d // 2)]),
                "axes": rng.choice([2, 3, 3, 4]), "order": rng.choice(["blocks", "turn"]), "layout": rng.choice(["half", "pairs"]),
                "dtype": dtype, "store": store}
        if store:
            case |= {"codes": codes, "page": page, "out": dtype if dtype != "f32" else rng.choice(["bf16", "f16"])}
        return case
    if kind == "verify":
        b, tree, vocab = _log(rng, 1, 64), rng.random() < 0.6, _log(rng, *VOCAB)
        t = _log(rng, 1, 64) if tree else _log(rng, 1, 17)
        while b * t * vocab > MAX_PROBS:
            if b > 1:
                b = (b + 1) // 2
            else:
                vocab = (vocab + 1) // 2
        return {"kind": kind, "b": b, "t": t, "vocab": vocab, "tree": tree, "draft": rng.random() < 0.5,
                "width": rng.choice([2, 3, 4]) if tree else 1, "dtype": dtype, "ragged": rng.random() < 0.6}
    do, b, l = rng.choice(["keep", "fork"]), _log(rng, 1, 64), _log(rng, 1, 8192)
    t, n = _log(rng, 1, 64), _log(rng, 1, 128)
    l = max(l, t)
    while (b * (l + t + page) + n * (t + 2 * page)) * hk * 128 > MAX_CACHE:
        if b > 1:
            b = (b + 1) // 2
        elif n > 1:
            n = (n + 1) // 2
        else:
            l = t = (l + 1) // 2
    return {"kind": kind, "do": do, "codes": codes, "b": b, "l": l, "t": t, "hk": hk, "d": d, "page": page,
            "n": n if do == "fork" else 0}


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ geometry
def _new(case):
    """New tokens of each sequence: those of a ragged batch differ."""
    t = case["t"]
    return [max(1, t - (i * 37 % 11) * t // 16) if case.get("ragged") else t for i in range(case["b"])]


def _lengths(case):
    """Cached tokens of each sequence, ragged down to a quarter, never fewer than the new ones."""
    l, t = case["l"], case["t"]
    return [max(t, l - (l * 3 // 4) * (i * 61 % 97) // 97) for i in range(case["b"])]


def _axes(case):
    """The axis of each plane: blocks of about one size (the last one larger), or one plane of each in turn."""
    half, axes = case["r"] // 2, case["axes"]
    if case["order"] == "turn":
        return [i % axes for i in range(half)]
    return [min(i // max(half // axes, 1), axes - 1) for i in range(half)]


def _frequencies(case):
    return 10000.0 ** (-torch.arange(0, case["r"], 2, dtype=torch.float64) / case["r"])


def _padded(d):
    return (d + 31) // 32 * 32


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 31)
    return g


def _normal(g, shape, std=1.0, dtype="f32"):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(_TYPES[dtype])


def _stored(g, case, pages):
    """Codes and scales of a cache in use."""
    shape = (pages, case["hk"], case["page"])
    c = torch.randint(-127, 128, (*shape, _padded(case["d"])), generator=g, device="cuda", dtype=torch.int8)
    if case["codes"] == "fp8":
        c = (c.float() * 3.5).to(torch.float8_e4m3fn).view(torch.uint8)
    c[..., case["d"]:] = 0
    return c, torch.rand(shape, generator=g, device="cuda") * 0.02 + 0.01


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def _prepare_adapt(case, g, rng):
    m, count, r, parts, k, n = (case[f] for f in ("m", "count", "r", "parts", "k", "n"))
    if case["rows"] == "mixed":  # one row of eight has no adapter
        index = [rng.randrange(count) if m == 1 or rng.random() < 0.875 else -1 for _ in range(m)]
    else:  # prompts of differing length, one after the other
        edges = sorted(rng.randrange(m) for _ in range(min(count, m) - 1)) + [m]
        owners, index = rng.sample(range(-1, count), len(edges)), []
        for edge, owner in zip(edges, owners):
            index += [owner] * (edge - len(index))
    return {"case": case, "x": _normal(g, (m, k), 1.0, case["dtype"]), "y": _normal(g, (m, n)),
            "a": _normal(g, (count, parts, r, k), k ** -0.5, case["weights"]),
            "b": _normal(g, (count, n, r), r ** -0.5, case["weights"]),
            "scales": torch.rand(count, generator=g, device="cuda") + 0.5, "index": _ints(index),
            "most": max(index.count(i) for i in set(index))}


def _prepare_turn(case, g, rng):
    n, d, axes = case["n"], case["d"], case["axes"]
    side = max(1, math.isqrt(n))
    i = torch.arange(n, device="cuda")
    start = rng.randrange(1, 4096)
    if n < 64:  # streams, each somewhere else
        pos = torch.randint(1, 8192, (axes, n), generator=g, device="cuda")
    else:  # the patches of an image, row by row (and frame by frame)
        pos = torch.stack([start + i // (side * side), start + i // side % side, start + i % side, start + i][:axes])
    s = {"case": case, "q": _normal(g, (n, case["h"], d), 1.0, case["dtype"]), "k": _normal(g, (n, case["hk"], d), 1.0, case["dtype"]),
         "positions": pos, "frequencies": _frequencies(case).cuda(), "axis": torch.tensor(_axes(case)).cuda()}
    if case["store"]:
        b = n if n < 64 else 1  # up to 63 tokens: a sequence each; more: one prompt
        per = (n // b + case["page"] - 1) // case["page"]
        s["v"] = _normal(g, (n, case["hk"], d), 0.7, case["dtype"])
        s["k_cache"], s["k_scale"] = _stored(g, case, max(b * per + 3, 8))
        s["v_cache"], s["v_scale"] = _stored(g, case, max(b * per + 3, 8))
        s["table"] = torch.randperm(b * per, generator=g, device="cuda").view(b, per).to(torch.int32)
        s["lengths"] = _ints([n // b] * b)
    return s


def _parents(rng, t, width):
    """A tree of t tokens: each one's parent, before it and among the last dozen, none with more than `width` children."""
    parents, children = [-1], [0] * t
    for i in range(1, t):
        p = rng.choice([j for j in range(max(0, i - 12), i) if children[j] < width] or [i - 1])
        children[p] += 1
        parents.append(p)
    return parents


def _prepare_verify(case, g, rng):
    new, vocab = _new(case), case["vocab"]
    offsets = _starts(new)
    rows = offsets[-1]
    parents = [p for t in new for p in (_parents(rng, t, case["width"]) if case["tree"] else range(-1, t - 1))]
    first = [offsets[i] for i, t in enumerate(new) for _ in range(t)]
    rank, seen = [], {}
    for i, p in enumerate(parents):  # the how manieth child
        rank.append(seen.get((first[i], p), 0))
        seen[(first[i], p)] = rank[-1] + 1
    up = torch.tensor([f + max(p, 0) for f, p in zip(first, parents)]).cuda()
    z = torch.randn(rows, vocab, generator=g, device="cuda") * 3.5
    target = torch.softmax(z, 1).to(_TYPES[case["dtype"]])
    z += torch.randn(rows, vocab, generator=g, device="cuda")
    if case["draft"]:  # drawn from the draft model's probabilities after the parent
        draft = torch.softmax(z, 1).to(_TYPES[case["dtype"]])
        noise = torch.rand(rows, vocab, generator=g, device="cuda").clamp_min_(1e-30).log_().neg_()
        tokens = (draft.float()[up] / noise).argmax(1)
    else:  # its likeliest ones
        draft = None
        tokens = z.topk(max(rank) + 1, 1).indices[up, torch.tensor(rank).cuda()]
    tree = torch.zeros(case["b"], case["t"], case["t"], dtype=torch.bool)
    for i, t in enumerate(new):  # what the attention over the tree had: each token's line up to itself
        for j in range(t):
            p = parents[offsets[i] + j]
            if p >= 0:
                tree[i, j] = tree[i, p]
            tree[i, j, j] = True
    return {"case": case, "tokens": tokens, "target": target, "draft": draft, "parents": _ints(parents), "offsets": _ints(offsets),
            "tree": tree.cuda(), "rows": rows, "accept": torch.rand(rows, generator=g, device="cuda"),
            "final": torch.rand(case["b"], generator=g, device="cuda"), "table": _ints([[0]] * case["b"]), "lengths": _ints(new)}


def _prepare_pages(case, g, rng):
    lengths, b, t, page = _lengths(case), case["b"], case["t"], case["page"]
    per = max((v + t + page - 1) // page for v in lengths)
    held = [(v + page - 1) // page for v in lengths]
    pages = (b * per + case["n"] * (t // page + 2) + 5) * 9 // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda")
    table = order[:b * per].view(b, per).to(torch.int32)
    s = {"case": case, "lengths": _ints(lengths), "pages": pages}
    s["k_cache"], s["k_scale"] = _stored(g, case, pages)
    s["v_cache"], s["v_scale"] = _stored(g, case, pages)
    if case["do"] == "keep":
        # the root, perhaps its likeliest line, then branches further behind
        paths, kept = torch.full((b, t), -1, dtype=torch.int32), []
        for i in range(b):
            n = rng.randint(1, max(1, min(8, (t + 1) // 2)))
            line = rng.randint(1, n)
            rows = list(range(line)) + sorted(rng.sample(range(n, t), n - line))
            paths[i, :n] = torch.tensor(rows, dtype=torch.int32)
            kept.append(n)
        return s | {"table": table, "path": paths.cuda(), "kept": _ints(kept)}
    used = torch.arange(per, device="cuda")[None] < torch.tensor(held).cuda()[:, None]
    holders = torch.zeros(pages, dtype=torch.int32, device="cuda")
    holders[order[:b * per].view(b, per)[used]] = 1
    holders[order[-(pages // 9):]] = 2  # other requests'
    parents = [i * b // case["n"] for i in range(case["n"])]
    rng.shuffle(parents)
    s |= {"table": torch.where(used, table, -1).contiguous(), "holders": holders, "parents": _ints(parents)}
    s["grown"] = s["lengths"][s["parents"].long()] + t
    return s


def prepare(case, seed):
    g, rng = _gen(seed), random.Random(int(seed) * 7 + 5)
    return {"adapt": _prepare_adapt, "turn": _prepare_turn, "verify": _prepare_verify, "pages": _prepare_pages}[case["kind"]](case, g, rng)


# ------------------------------------------------------------------ the plain forms
def _plain_adapt(s):
    """Rows gathered by their adapter, two products for all adapters at once, and back."""
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    count, parts, r, k = a.shape
    m, n, most = x.shape[0], b.shape[1], s["most"]
    group = torch.where(s["index"] < 0, count, s["index"]).long()  # rows without one last
    mine = group[:, None] == torch.arange(count + 1, device="cuda")
    place = mine.int().cumsum(0).gather(1, group[:, None])[:, 0] - 1
    xs = torch.zeros(count + 1, most, k, device="cuda")
    xs[group, place] = x
    low = torch.bmm(xs[:count], a.view(count, parts * r, k).transpose(1, 2).contiguous())
    low = low.view(count, most, parts, r).transpose(1, 2).reshape(count * parts, most, r)
    up = torch.bmm(low, b.view(count * parts, n // parts, r).transpose(1, 2).contiguous())
    up = up.view(count, parts, most, n // parts).transpose(1, 2).reshape(count, most, n) * s["scales"][:, None, None]
    up = torch.cat([up, torch.zeros(1, most, n, device="cuda")])
    return s["y"] + up[group, place]


def _turned(x, s):
    case = s["case"]
    a = s["positions"].double()[s["axis"]].t() * s["frequencies"]  # far positions lose their angle in 32 bits
    c, n = a.cos().float()[:, None], a.sin().float()[:, None]
    r, v = case["r"], x.float()
    if case["layout"] == "half":
        p, q = v[..., :r // 2], v[..., r // 2:r]
        turned = torch.cat([p * c - q * n, q * c + p * n], -1)
    else:
        p, q = v[..., 0:r:2], v[..., 1:r:2]
        turned = torch.stack([p * c - q * n, q * c + p * n], -1).flatten(-2)
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


def _plain_turn(s):
    case = s["case"]
    q, k = _turned(s["q"], s), _turned(s["k"], s)
    if not case["store"]:
        return q.to(s["q"].dtype), k.to(s["k"].dtype)
    b, n, page, d = s["table"].shape[0], case["n"], case["page"], case["d"]
    row = torch.arange(n, device="cuda")
    pos = row % (n // b)
    pages, off = s["table"][row // (n // b), pos // page].long(), pos % page
    (kc, ks), (vc, vs) = _coded(k, case["codes"]), _coded(s["v"].float(), case["codes"])
    s["k_cache"][pages, :, off, :d], s["k_scale"][pages, :, off] = kc, ks
    s["v_cache"][pages, :, off, :d], s["v_scale"][pages, :, off] = vc, vs
    out = _TYPES[case["out"]]
    back = [(_floats(c[pages, :, off, :d]) * x[pages, :, off][..., None]).to(out)
            for c, x in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
    return [q.to(s["q"].dtype), *back]


def _plain_verify(s):
    """All tokens of all trees at once: each one's test against what its earlier siblings leave, in 64 bits."""
    case, off = s["case"], s["offsets"].long()
    b, most, vocab = case["b"], case["t"], case["vocab"]
    t = torch.arange(most, device="cuda")
    live = t[None] < (off[1:] - off[:-1])[:, None]
    rows = (off[:-1, None] + t).clamp_max(s["rows"] - 1)  # [b, most]
    parents = torch.where(live & (t[None] > 0), s["parents"][rows].long(), -1)
    tokens = torch.where(live, s["tokens"][rows], -1)
    up = rows.gather(1, parents.clamp_min(0))
    u = s["accept"][rows].double()
    sibling = (parents[:, :, None] == parents[:, None]) & (parents >= 0)[:, :, None]  # [b, child, other]
    earlier = sibling & (t[None, :, None] > t)
    p = s["target"][up, tokens.clamp_min(0)].double()
    if s["draft"] is None:
        again = (earlier & (tokens[:, :, None] == tokens[:, None])).any(2)
        p = torch.where(again, 0.0, p)
        accepted = u * (1.0 - torch.where(earlier, p[:, None], 0.0).sum(2)) < p
    else:
        q, nth = s["draft"][up, tokens.clamp_min(0)].double(), earlier.sum(2)
        target, draft = s["target"].double(), s["draft"].double()
        shares, mass, share = [torch.zeros(s["rows"], dtype=torch.float64, device="cuda")], [], torch.ones(s["rows"], dtype=torch.float64, device="cuda")
        mass.append(share)
        for _ in range(case["width"]):  # what is left after each child that is turned down
            shares.append(shares[-1] + mass[-1])
            mass.append(torch.addcmul(target, draft, -shares[-1][:, None]).clamp_min_(0.0).sum(1))
        shares, mass = torch.stack(shares), torch.stack(mass)
        accepted = u * q * mass[nth, up] < p - shares[nth, up] * q
    accepted &= parents >= 0
    chosen = accepted & ~(earlier & accepted[:, None]).any(2)  # the first of its siblings
    chosen |= t[None] == 0
    on = live & ~(s["tree"] & ~chosen[:, None]).any(2)
    kept = on.sum(1)
    last = torch.where(on, t[None], 0).amax(1)
    path = torch.where(on, t[None], most).sort(1).values
    path = torch.where(path < most, path, -1)
    tried = (parents == last[:, None]) & live  # its children, all turned down
    at = rows.gather(1, last[:, None])[:, 0]
    left = s["target"][at].double()
    if s["draft"] is None:
        gone = torch.zeros(b, vocab + 1, device="cuda").scatter_(1, torch.where(tried, tokens, vocab), 1.0)
        rest = torch.where(gone[:, :vocab] > 0, 0.0, left)
    else:
        rest = (left - shares[tried.sum(1), at][:, None] * s["draft"][at].double()).clamp_min_(0.0)
    left = torch.where(rest.sum(1, keepdim=True) > 0, rest, left)  # where nothing is left, the target's own
    sums = left.cumsum(1)
    goal = s["final"].double()[:, None] * sums[:, -1:]
    following = (sums <= goal).sum(1).clamp_max(vocab - 1)
    return {"path": path.int(), "kept": kept.int(), "next": following}


def _buffers(s):
    return {name: s[name] for name in ("k_cache", "k_scale", "v_cache", "v_scale")}


def _plain_keep(s):
    case, page, path = s["case"], s["case"]["page"], s["path"].long()
    start = s["lengths"].long() - case["t"]
    i = torch.arange(path.shape[1], device="cuda")
    moved = i[None] < s["kept"][:, None]
    b = torch.arange(path.shape[0], device="cuda")[:, None]
    src, dst = (start[:, None] + torch.where(moved, v, 0) for v in (path, i[None]))  # others: the root onto itself
    sp, so, dp, do = s["table"][b, src // page].long(), src % page, s["table"][b, dst // page].long(), dst % page
    for buffer in _buffers(s).values():
        buffer[dp, :, do] = buffer[sp, :, so]
    return _buffers(s) | {"lengths": (start + s["kept"]).int()}


def _plain_fork(s):
    page, holders, par = s["case"]["page"], s["holders"], s["parents"].long()
    lengths, rows = s["lengths"].long()[par], s["table"][par]
    i = torch.arange(rows.shape[1], device="cuda")[None]

    def hold(entries, by):
        holders.scatter_add_(0, entries.clamp_min(0).flatten().long(), ((entries >= 0).int() * by).flatten())

    def take(wanted):
        """The lowest free pages, in order, for the wanted places."""
        free = torch.sort((holders > 0).int(), stable=True).indices
        got = torch.where(wanted, free[(wanted.flatten().int().cumsum(0) - 1).clamp_min(0).view(wanted.shape)].int(), -1)
        hold(got, 1)
        return got

    whole = (lengths // page)[:, None]
    children = torch.where(i < whole, rows, -1)
    hold(children, 1)
    begun = lengths % page > 0
    target = take(begun)
    source = torch.where(begun, rows.gather(1, whole.clamp_max(rows.shape[1] - 1))[:, 0], -1)
    children = torch.where((i == whole) & begun[:, None], target[:, None], children)
    src, dst = (torch.where(begun, v, rows[:, 0]).long() for v in (source, target))  # others: their first page onto itself
    for buffer in _buffers(s).values():
        buffer[dst] = buffer[src]
    grown = (s["grown"].long()[:, None] + page - 1) // page
    children = torch.where((children < 0) & (i < grown), take((children < 0) & (i < grown)), children)
    hold(children, -1)
    return _buffers(s) | {"children": children, "source": source, "target": target, "holders": holders}


# ------------------------------------------------------------------ the framework's calls
def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neo-theano_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import theano_quantize

    return theano_quantize


def _own_run(s):
    tq, case = _framework(), s["case"]
    if case["kind"] == "adapt":
        if "adapters" not in s:  # loaded once, as the layer's weights are
            s["adapters"] = tq.Adapters(s["a"], s["b"], s["scales"])
        return s["adapters"].add(s["x"], s["index"], s["y"])
    if case["kind"] == "turn":
        rotary = tq.Rotary(s["frequencies"], case["layout"] == "pairs", axes=_axes(case))
        if not case["store"]:
            return rotary.apply(s["q"], s["k"], s["positions"])
        cache = tq.KVCache(s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], case["d"])
        new = tq.KVBatch(s["table"], s["lengths"], case["n"] // s["table"].shape[0])
        return [cache.write_rotary(s["q"], s["k"], s["v"], rotary, new, s["positions"]), *cache.read(new, _TYPES[case["out"]])]
    if case["kind"] == "verify":
        new = tq.KVBatch(s["table"], s["lengths"], case["t"], s["offsets"], s["rows"])
        path, kept, following = tq.verify_drafts(s["tokens"], s["target"], new, s["accept"], s["final"], draft=s["draft"],
                                                 parents=s["parents"] if case["tree"] else None)
        return {"path": path, "kept": kept, "next": following}
    cache = tq.KVCache(s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], case["d"])
    if case["do"] == "keep":
        return _buffers(s) | {"lengths": cache.keep(tq.KVBatch(s["table"], s["lengths"], case["t"]), s["path"], s["kept"])}
    pool = tq.PagePool(s["holders"], case["page"])
    children, source, target = pool.fork(s["table"], s["lengths"], s["parents"])
    cache.copy_pages(source, target)
    pool.grow(children, s["grown"])
    had = children.clone()
    pool.free(children)
    return _buffers(s) | {"children": had, "source": source, "target": target, "holders": s["holders"]}


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["kind"] == "pages":
        return _plain_keep(state) if case["do"] == "keep" else _plain_fork(state)
    return {"adapt": _plain_adapt, "turn": _plain_turn, "verify": _plain_verify}[case["kind"]](state)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_adapt(s):
    y, index = s["y"].double(), s["index"].tolist()
    parts, n = s["case"]["parts"], s["case"]["n"]
    for i in sorted(set(index) - {-1}):
        rows = torch.tensor([j for j, v in enumerate(index) if v == i], device="cuda")
        x = s["x"][rows].double()
        for p in range(parts):
            cols = slice(p * n // parts, (p + 1) * n // parts)
            y[rows, cols] += (x @ s["a"][i, p].double().t().contiguous()) @ s["b"][i, cols].double().t().contiguous() * float(s["scales"][i])
    return y


def _rotate64(x, s):
    """Complex numbers times e^(i angle)."""
    case, x = s["case"], x.double()
    r = case["r"]
    angle = torch.stack([s["positions"][a].double() * f for a, f in zip(_axes(case), _frequencies(case).tolist())], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if case["layout"] == "half":
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., r:]], -1)
    z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1)


def _value64(x, kind):
    """What a token's head is stored as: its scale is a 32-bit number by definition, the FP8 quotient too."""
    s = (x.abs().amax(-1, keepdim=True) / (127.0 if kind == "i8" else 448.0)).clamp_min(1e-10).float().double()
    if kind == "i8":
        v = x / s
        return torch.sign(v) * (v.abs() + 0.5).floor() * s
    v = (x / s).float().double().clamp(-448, 448)
    step = torch.exp2(torch.frexp(v.abs().clamp_min(2.0 ** -6))[1].double() - 4)
    return (v / step).round() * step * s


def _exact_verify(s):
    """One tree after the other, one child after the other."""
    off, out = s["offsets"].tolist(), {"path": [], "kept": [], "next": []}
    parents, tokens, accept, final = (s[n].tolist() for n in ("parents", "tokens", "accept", "final"))
    for b in range(len(off) - 1):
        node, path, gone = 0, [0], []
        p = s["target"][off[b]].double()
        q, share, mass = None if s["draft"] is None else s["draft"][off[b]].double(), 0.0, 1.0
        left = p.clone()
        for t in range(1, off[b + 1] - off[b]):
            r = off[b] + t
            if parents[r] != node:
                continue
            x = tokens[r]
            if accept[r] * (1.0 if q is None else float(q[x])) * mass < float(left[x] if share == 0.0 else p[x] - share * q[x]):
                node, gone = t, []
                path.append(t)
                p = s["target"][r].double()
                q, share, mass = None if s["draft"] is None else s["draft"][r].double(), 0.0, 1.0
                left = p.clone()
            elif q is None:
                mass -= float(left[x])
                left[x] = 0.0
            else:
                share += mass
                left = (p - share * q).clamp_min(0.0)
                mass = float(left.sum())
        sums = left.cumsum(0)
        out["path"].append(path + [-1] * (s["case"]["t"] - len(path)))
        out["kept"].append(len(path))
        out["next"].append(min(int((sums <= final[b] * sums[-1]).sum()), len(p) - 1))
    return {"path": _ints(out["path"]), "kept": _ints(out["kept"]), "next": torch.tensor(out["next"]).cuda()}


def _exact_keep(s):
    page, t, table, lengths, paths, kept = s["case"]["page"], s["case"]["t"], *(s[n].tolist() for n in ("table", "lengths", "path", "kept"))
    for buffer in _buffers(s).values():
        before = buffer.clone()
        for b, n in enumerate(kept):
            for i in range(n):
                src, dst = lengths[b] - t + paths[b][i], lengths[b] - t + i
                buffer[table[b][dst // page], :, dst % page] = before[table[b][src // page], :, src % page]
    return _buffers(s) | {"lengths": _ints([v - t + n for v, n in zip(lengths, kept)])}


def _exact_fork(s):
    page, table, lengths, parents, grown = s["case"]["page"], *(s[n].tolist() for n in ("table", "lengths", "parents", "grown"))
    holders = s["holders"].tolist()
    children, source, target = [], [], []
    for p in parents:
        children.append(table[p][:lengths[p] // page] + [-1] * (len(table[p]) - lengths[p] // page))
        for e in children[-1]:
            if e >= 0:
                holders[e] += 1

    def take():
        e = holders.index(0)
        holders[e] = 1
        return e

    for c, p in enumerate(parents):
        begun = lengths[p] % page > 0
        source.append(table[p][lengths[p] // page] if begun else -1)
        target.append(take() if begun else -1)
        if begun:
            children[c][lengths[p] // page] = target[-1]
            for buffer in _buffers(s).values():
                buffer[target[-1]] = buffer[source[-1]]
    for c, n in enumerate(grown):
        for i in range((n + page - 1) // page):
            if children[c][i] < 0:
                children[c][i] = take()
    return _buffers(s) | {"children": _ints(children), "source": _ints(source), "target": _ints(target), "holders": s["holders"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "turn":
        q, k = _rotate64(s["q"], s), _rotate64(s["k"], s)
        return [q, _value64(k, case["codes"]), _value64(s["v"].double(), case["codes"])] if case["store"] else (q, k)
    if case["kind"] == "pages":
        return _exact_keep(s) if case["do"] == "keep" else _exact_fork(s)
    return {"adapt": _exact_adapt, "verify": _exact_verify}[case["kind"]](s)


# ------------------------------------------------------------------ the work
def work(case):
    kind = case["kind"]
    if kind == "adapt":
        m, r, k, n, parts = (case[f] for f in ("m", "r", "k", "n", "parts"))
        used = min(case["count"], m)  # adapters that rows name
        return {"bytes": m * (k * _SIZE[case["dtype"]] + 8 * n + 4) + used * r * (parts * k + n) * 2, "flops": 2 * m * r * (parts * k + n)}
    if kind == "turn":
        n, d, heads, size = case["n"], case["d"], case["h"] + case["hk"], _SIZE[case["dtype"]]
        moved = 2 * n * heads * d * size + 8 * n * case["axes"]
        if case["store"]:  # k leaves as codes, v comes and leaves as codes, and both come back
            moved += n * case["hk"] * (4 * (d + 4) + 2 * d * _SIZE[case["out"]])
        return {"bytes": moved, "flops": 3 * n * heads * case["r"]}
    if kind == "verify":
        rows = sum(_new(case))
        models = 2 if case["draft"] else 1
        # of each sequence one row of what is left, and two numbers for each drafted token
        return {"bytes": (case["b"] * case["vocab"] + rows) * models * _SIZE[case["dtype"]] + 16 * rows,
                "flops": 3 * case["b"] * case["vocab"] * models}
    row = case["hk"] * (_padded(case["d"]) + 4) * 2  # a token's keys and values
    if case["do"] == "keep":
        n = case["b"] * min(4, case["t"])  # about so many stay
        return {"bytes": 2 * n * row + 8 * case["b"] * (case["t"] + 3), "flops": 0}
    per = (max(_lengths(case)) + case["t"] + case["page"] - 1) // case["page"]
    return {"bytes": 2 * case["n"] * case["page"] * row + 8 * case["n"] * per, "flops": 0}
