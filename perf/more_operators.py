"""The 8-bit decoder's operators, as cases that can be timed and checked: a step's products, its cache and the
token it draws.

A case is a dict of plain values. ``listed()`` gives the standing ones and ``draw(rng)`` one more of the same
ranges; ``prepare(case, seed)`` makes what a program has in hand before the call, ``run(state)`` makes one pass
and returns its outputs (with ``own`` false by elementary torch operations, with ``own`` true by the
framework's calls), ``exact(case, seed)`` gives the same outputs in 64 bits, and ``work(case)`` the bytes and
operations that the pass cannot do without.

The kinds of case:

product  rows times weights in 8-bit floating point (e4m3) with a scale for each block of 128 x 128; the rows
         are rounded to e4m3 in groups of 128, each with the least power of two that holds its largest value
         (``Kernels.linear_e4m3_device``)
paged    a chunk of new tokens, or a single one, of each sequence over pages of e4m3 values whose blocks of
         tokens have a power of two for each head (``Attention.paged``)
append   new keys, rotated, and values into such pages (``PagedCache.append``)
sample   a token of each row of logits, from given random numbers, by temperature, top-k, top-p and min-p
         (``Sampler.sample``)

750 rows are a minute of audio at 12.5 frames per second, 640 the TDT decoder's width, 8198 its joint's
outputs; the other sizes are generic. Rows are N(0, 1)."""
import math

import numpy as np
import torch

own = False

GROUP = 128  # inputs of a product that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
E4M3 = torch.float8_e4m3fn
LOWEST = -100  # the least exponent of a scale


# ------------------------------------------------------------------------------------------ cases

def _product(**kw):
    case = {"kind": "product", "type": "f32", "to": "f32", "m": 1, "k": 4096, "n": 4096, "pad": 0, "bias": True,
            "act": "none", "scale": 1.0}
    case.update(kw)
    return case


def _paged(**kw):
    case = {"kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "d": 128, "sequences": 32, "new": 1,
            "ragged": True, "cached": 8192, "page": 16, "block": 16, "cap": 0.0, "left": -1, "prefix": 0, "slopes": False}
    case.update(kw)
    return case


def _append(**kw):
    case = {"kind": "append", "type": "f32", "sequences": 4, "new": 2047, "kv_heads": 8, "d": 128, "dim": 128,
            "interleaved": False, "cached": 2560, "page": 16, "block": 16}
    case.update(kw)
    return case


def _sample(**kw):
    case = {"kind": "sample", "type": "f32", "rows": 1, "n": 8198, "temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.0,
            "mixed": False, "spread": 2.5, "shut": 0.05}
    case.update(kw)
    return case


def listed():
    return [
        # One stream's token through a decoder's narrow gates: the smallest product, where latency counts.
        dict(_product(m=1, k=640, n=2560), name="product, 1 x 640 -> 2560"),
        # A server's decode step, sixteen streams through a wide feed-forward layer: bound by the weights.
        dict(_product(type="bf16", m=16, k=4096, n=16384, bias=False, act="silu"), name="product, 16 x 4096 -> 16384"),
        # A minute of audio through an encoder's feed-forward layer: the ordinary product.
        dict(_product(m=750, k=1024, n=4096, act="silu"), name="product, 750 x 1024 -> 4096"),
        # A long batch of prompts through a wide layer, 16-bit rows in and out: bound by the matrix cores.
        dict(_product(type="bf16", to="bf16", m=8192, k=8192, n=8192, bias=False), name="product, 8192^3"),
        # Eight streams, one f32 frame each over a minute of frames before it: the smallest attention.
        dict(_paged(type="f32", heads=8, kv_heads=8, sequences=8, cached=750, page=25, block=25), name="one token, 8 streams"),
        # A server's decode step over long caches.
        dict(_paged(), name="one token, 32 x 8192"),
        # A chunk of a long prompt over what is cached of it.
        dict(_paged(sequences=1, new=509, cached=32768, page=64, block=32, ragged=False), name="chunk of 509 over 32768"),
        # One token's keys and values of each of eight streams: the smallest append.
        dict(_append(sequences=8, new=1, cached=750, page=25, block=25), name="append, 8 tokens"),
        # Four prompts' keys and values, each stopping inside a block.
        dict(_append(), name="append, 4 x 2047"),
        # One stream's token from the joint's outputs: the smallest draw.
        dict(_sample(top_k=50, top_p=0.95), name="sample, 1 x 8198"),
        # A batch of requests, each with options of its own.
        dict(_sample(rows=48, n=50000, mixed=True), name="sample, 48 x 50000"),
        # A large batch over a large vocabulary, most of whose mass takes part.
        dict(_sample(rows=256, n=131072, temperature=1.0, top_p=0.9, min_p=0.0001), name="sample, 256 x 131072"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "paged", "paged", "paged", "append", "append", "sample", "sample"])
    if kind == "product":
        m, k = _log(rng, 1, 4000), _log(rng, 16, 8192)
        if rng.random() < 0.5:
            k = -(-k // GROUP) * GROUP
        return _product(type=rng.choice(["f32", "f32", "f16", "bf16"]), to=rng.choice(["f32", "f32", "f16", "bf16"]), m=m, k=k,
                        n=_log(rng, 16, 8192), pad=rng.choice([0, 0, 8, 3]), bias=rng.random() < 0.5,
                        act=rng.choice(["none", "relu", "silu"]), scale=rng.choice([1.0, 0.5]))
    if kind == "paged":
        kv = rng.choice([1, 2, 4, 8])
        sequences = rng.choice([1, 1, 3, 8, 17])
        new = rng.choice([1, 1, 2, 5, _log(rng, 8, 300)])
        page, block = rng.choice([(1, 1), (7, 7), (16, 16), (16, 8), (64, 16), (64, 64), (256, 1), (256, 128)])
        return _paged(type=rng.choice(["f16", "bf16", "f32"]), heads=kv * rng.choice([1, 2, 4, 6]), kv_heads=kv,
                      d=rng.choice([64, 96, 128, 128, 256]), sequences=sequences, new=new,
                      cached=_log(rng, new + 1, 24000 // sequences), page=page, block=block,
                      cap=rng.choice([0.0, 0.0, 40.0]), left=rng.choice([-1, -1, 200]), prefix=rng.choice([0, 0, 4]),
                      slopes=rng.random() < 0.25)
    if kind == "append":
        d = rng.choice([64, 128, 256])
        sequences = rng.choice([1, 3, 8, 20])
        new = _log(rng, 1, 4000 // sequences)
        page, block = rng.choice([(1, 1), (7, 7), (16, 16), (16, 4), (64, 32), (256, 256)])
        return _append(type=rng.choice(["f32", "bf16", "f16"]), sequences=sequences, new=new, kv_heads=rng.choice([1, 2, 8]),
                       d=d, dim=rng.choice([0, d, d // 2]), interleaved=rng.random() < 0.5,
                       cached=new + _log(rng, 1, 2000), page=page, block=block)
    n = _log(rng, 2, 131072)
    return _sample(type=rng.choice(["f32", "f32", "f16", "bf16"]), rows=_log(rng, 1, max(1, min(256, (1 << 23) // n))), n=n,
                   temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                   top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.2]),
                   mixed=rng.random() < 0.3, spread=rng.choice([0.5, 2.5, 6.0]), shut=rng.choice([0.0, 0.05, 0.9]))


# ------------------------------------------------------------------------------- inputs from a seed

_stream = None


def _own_stream():
    """The program's one stream, torch's current stream from the first call on."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    torch.cuda.set_stream(_stream)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _shapes(case, seed):
    """The ragged sizes that the seed decides, on the host."""
    rng = np.random.default_rng([int(seed), 17])
    n, new, cached = case["sequences"], case["new"], case["cached"]
    news, lens = [new] * n, [cached] * n
    if case.get("ragged", True):
        counts = np.random.default_rng([n, new])  # the outputs' sizes are the case's, whatever the seed
        news = [new] + counts.integers(1, new + 1, n - 1).tolist()
        lens = [cached] + [int(rng.integers(m, cached + 1)) for m in news[1:]]
    width = -(-cached // case["page"])
    pages = n * width + 3  # some pages belong to others
    tables = rng.permutation(pages)[:n * width].reshape(n, width)
    return {"new": news, "lens": lens, "tables": tables, "pages": pages}


def _least_exponent(top):
    """The least e with top <= 448 2^e, from LOWEST on, of finite values."""
    part, e = torch.frexp(top)  # top = part 2^e with part in [1/2, 1), and 448 = 7/8 2^9
    return torch.where(top > 0, e - 9 + (part > 0.875).int(), torch.full_like(e, LOWEST)).clamp(min=LOWEST)


def _two_to(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _pages(case, pages, gen):
    """Pages [pages, page, kv_heads, d] of values as a model's keys have them, sizes differing from block to block,
    rounded to e4m3, and their blocks' exponents."""
    page, block, kv, d = case["page"], case["block"], case["kv_heads"], case["d"]
    x = torch.randn((pages, page // block, block, kv, d), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((pages, page // block, 1, kv, 1), generator=gen, device="cuda"))
    e = _least_exponent(x.abs().amax((2, 4)))
    x *= _two_to(-e)[:, :, None, :, None]
    return x.to(E4M3).view(pages, page, kv, d), e.to(torch.int8)


def prepare(case, seed):
    _own_stream()
    kind = case["kind"]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 31)

    def normal(*shape, type="f32"):
        return torch.randn(shape, generator=gen, device="cuda").to(TYPES[type])

    s = {"case": case}
    if kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        s["a"] = normal(m, k + case["pad"], type=case["type"])[:, :k]
        # A checkpoint's weights: the values of each block over its largest's 448th.
        nb, kb = -(-n // GROUP), -(-k // GROUP)
        w = torch.zeros((nb * GROUP, kb * GROUP), device="cuda")
        w[:n, :k] = normal(n, k) / math.sqrt(k)
        w = w.view(nb, GROUP, kb, GROUP)
        s["scales"] = w.abs().amax((1, 3)) / 448.0
        s["values"] = (w / s["scales"][:, None, :, None]).to(E4M3).view(nb * GROUP, kb * GROUP)[:n, :k].contiguous()
        s["bias"] = normal(n) if case["bias"] else None
        s["c"] = torch.empty((m, n), dtype=TYPES[case["to"]], device="cuda")
    elif kind in ("paged", "append"):
        shapes = _shapes(case, seed)
        kv, d = case["kv_heads"], case["d"]
        s["k"], s["k_exps"] = _pages(case, shapes["pages"], gen)
        s["v"], s["v_exps"] = _pages(case, shapes["pages"], gen)
        s["starts"], s["longest"] = _ints([0] + np.cumsum(shapes["new"]).tolist()), max(shapes["new"])
        s["lens"], s["tables"] = _ints(shapes["lens"]), _ints(shapes["tables"])
        rows = sum(shapes["new"])
        if kind == "paged":
            s["q"] = normal(rows, case["heads"], d, type=case["type"])
            s["out"] = torch.empty_like(s["q"])
            s["prefix"] = _ints([case["prefix"]] * case["sequences"]) if case["prefix"] else None
            if case["slopes"]:
                s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"])
        else:
            s["k_rows"], s["v_rows"] = normal(rows, kv, d, type=case["type"]), normal(rows, kv, d, type=case["type"])
    else:
        rows, n = case["rows"], case["n"]
        x = case["spread"] * normal(rows, n)
        x += 8.0 * (torch.rand((rows, n), generator=gen, device="cuda") < 3.0 / n)  # a few likely tokens
        x.masked_fill_(torch.rand((rows, n), generator=gen, device="cuda") < case["shut"], -math.inf)  # a grammar's mask
        s["logits"] = x.to(TYPES[case["type"]])
        s["uniforms"] = torch.rand(rows, generator=gen, device="cuda")
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["probs"] = torch.empty(rows, device="cuda")
        options = {name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")}
        if case["mixed"]:  # each request's own
            rng = np.random.default_rng([int(seed), 23])
            choices = {"temperature": [0.0, 0.3, 0.7, 1.0, 1.5], "top_k": [0, 1, 40, 1000], "top_p": [0.5, 0.9, 0.99, 1.0],
                       "min_p": [0.0, 0.02, 0.2]}
            for name, values in choices.items():
                kind_of = torch.int32 if name == "top_k" else torch.float32
                options[name] = torch.tensor(rng.choice(values, rows), dtype=kind_of, device="cuda")
        s["options"] = options
    return s


# --------------------------------------------------------------------------------- the plain forms

def _rounded(x, e):
    """x rounded to e4m3 under the exponents e."""
    return (x * _two_to(-e)).to(E4M3)


def _plain_product(s):
    c = s["case"]
    m, k, n = c["m"], c["k"], c["n"]
    kb = -(-k // GROUP)
    a = torch.zeros((m, kb * GROUP), device="cuda")
    a[:, :k] = s["a"]
    a = a.view(m, kb, GROUP)
    e = _least_exponent(a.abs().amax(2, keepdim=True))
    a = (_rounded(a, e).float() * _two_to(e)).view(m, kb * GROUP)[:, :k]
    w = s["values"].float() * s["scales"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    out = a @ w.t()
    if s["bias"] is not None:
        out = out + s["bias"]
    if c["act"] == "relu":
        out = out.clamp(min=0.0)
    elif c["act"] == "silu":
        out = out / (1.0 + torch.exp(-out))
    return (out * c["scale"]).to(s["c"].dtype)


def _values(s, name):
    """The pages' values in 32 bits, those of each sequence's positions [sequences, positions, kv_heads, d]."""
    c, tables = s["case"], s["tables"].long()
    x = s[name].view(torch.uint8)[tables].view(E4M3).float()
    scale = _two_to(s[name + "_exps"][tables].int()).repeat_interleave(c["block"], 2)
    return (x * scale[..., None]).flatten(1, 2)


def _plain_paged(s):
    c = s["case"]
    heads, kv, d, n, new = c["heads"], c["kv_heads"], c["d"], c["sequences"], s["longest"]
    lens, starts = s["lens"].long(), s["starts"].long()
    k, v = (_values(s, x)[:, :c["cached"]].permute(0, 2, 1, 3).unsqueeze(2) for x in ("k", "v"))
    counts = starts[1:] - starts[:-1]
    r, j = torch.arange(new, device="cuda"), torch.arange(k.shape[3], device="cuda")
    rows = (starts[:-1, None] + r).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(n, new, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
    distance = j - (lens[:, None, None] - counts[:, None, None] + r[:, None])
    shown = distance <= 0
    if c["left"] >= 0:
        shown = shown & (distance >= -c["left"])
    shown = ((shown | (j < c["prefix"])) & (j < lens[:, None, None]))[:, None, None]
    x = (q @ k.transpose(-1, -2)) * d ** -0.5
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if c["slopes"]:
        x = x - s["slopes"].view(kv, heads // kv, 1, 1) * distance.abs()[:, None, None]
    x = x.masked_fill(~shown, float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    out = (x @ v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, new, heads, d)
    return out[r < counts[:, None]].to(s["q"].dtype)


ROTARY_BASE = 10000.0


def _rotate(x, positions, case):
    """x [rows, heads, d] in 64 bits, its first dim values rotated by positions [rows]: what is rounded to eight bits next
    must lie on the right side of a border."""
    dim = case["dim"]
    if not dim:
        return x
    f = ROTARY_BASE ** (-2.0 * torch.arange(dim // 2, device="cuda", dtype=torch.float64) / dim)
    angle = positions.double()[:, None, None] * f
    cos, sin = torch.cos(angle), torch.sin(angle)
    turned, rest = x[..., :dim], x[..., dim:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        pair = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        pair = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([pair, rest], -1)


def _plain_append(s):
    c = s["case"]
    page, block, kv, d = c["page"], c["block"], c["kv_heads"], c["d"]
    starts, lens = s["starts"].long(), s["lens"].long()
    row = torch.arange(s["k_rows"].shape[0], device="cuda")
    which = torch.searchsorted(starts[1:], row, right=True)
    position = lens[which] - starts[which + 1] + row
    slot = s["tables"].long()[which, position // page] * page + position % page  # among all pages' rows
    at = slot // block  # among all blocks
    touched, of = torch.unique(at, return_inverse=True)
    older = torch.full_like(touched, block).scatter_reduce_(0, of, slot % block, "amin")  # rows of the block before the new ones
    for name, rows in (("k", _rotate(s["k_rows"].double(), position, c)), ("v", s["v_rows"])):
        rows = rows.float()
        values, exps = s[name].view(-1, block, kv, d), s[name + "_exps"].view(-1, kv)
        top = torch.zeros((touched.numel(), kv), device="cuda")
        top.scatter_reduce_(0, of[:, None].expand(-1, kv), rows.abs().amax(2), "amax")
        had, need = exps[touched].int(), _least_exponent(top)
        now = torch.where(older[:, None] > 0, torch.maximum(had, need), need)
        old = values.view(torch.uint8)[touched].view(E4M3)
        again = (torch.arange(block, device="cuda") < older[:, None])[:, :, None, None]
        old = torch.where(again, old.float() * _two_to(had - now)[:, None, :, None], old.float()).to(E4M3)
        values.view(torch.uint8)[touched] = old.view(torch.uint8)
        exps[touched] = now.to(torch.int8)
        s[name].view(-1, kv, d).view(torch.uint8)[slot] = _rounded(rows, now[of][..., None]).view(torch.uint8)
    return [s["k"], s["v"], s["k_exps"], s["v_exps"]]


def _plain_sample(s):
    options, n = s["options"], s["case"]["n"]
    t, top_k, top_p, min_p = (torch.as_tensor(options[x], device="cuda").to(torch.float32 if x != "top_k" else torch.int64)
                              .double().expand(s["tokens"].shape)[:, None] for x in ("temperature", "top_k", "top_p", "min_p"))
    x, index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    x = x.double()  # sums of many weights next to a border: 64 bits
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    place = torch.arange(n, device="cuda")
    most = torch.where(t > 0, torch.where(top_k > 0, top_k, torch.full_like(top_k, n)), torch.ones_like(top_k))
    w = torch.where(place < most, w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    kept = ((before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1)) & (w >= min_p) & (w > 0) | (place == 0)
    w = torch.where(kept, w, torch.zeros_like(w))
    sums = torch.cumsum(w, 1)
    # The first place whose sum passes the row's share; at most the last one kept.
    at = torch.minimum((sums <= s["uniforms"].double()[:, None] * sums[:, -1:]).sum(1), kept.sum(1) - 1)[:, None]
    none = ~(x[:, 0] > -math.inf)
    token = torch.where(none, torch.full_like(at[:, 0], -1), index.gather(1, at)[:, 0])
    prob = torch.where(none, torch.zeros_like(x[:, 0]), (w.gather(1, at) / sums[:, -1:])[:, 0])
    return [token.int(), prob.float()]


PLAIN = {"product": _plain_product, "paged": _plain_paged, "append": _plain_append, "sample": _plain_sample}


# ------------------------------------------------------------------------------ the framework's calls

_kept = {}


def _keep(key, make):
    """What a program makes once and keeps: its context, its operators' options."""
    if key not in _kept:
        _kept[key] = make()
    return _kept[key]


def _context():
    import telmo_amd

    return _keep("context", lambda: telmo_amd.Kernels(0, stream=_stream.cuda_stream))


def _workspace(want):
    """One workspace for all calls on the program's stream, as large as the largest wants it."""
    have = _kept.get("workspace")
    if have is None or have.numel() < want:
        have = _kept["workspace"] = torch.empty(max(want, 1 << 20), dtype=torch.uint8, device="cuda")
    return have


def _own_product(s):
    import telmo_amd

    c = s["case"]
    if "weights" not in s:  # laid out once, as a model is loaded
        s["weights"] = telmo_amd.E4m3Weights.from_device(_context(), s["values"], s["scales"])
        s["space"] = _workspace(s["weights"].workspace_bytes(c["m"]))
        s["epilogue"] = telmo_amd.Epilogue(bias=s["bias"], act=telmo_amd.Act[c["act"].upper()], scale=c["scale"])
    _context().linear_e4m3_device(s["a"], s["weights"], s["c"], s["epilogue"], workspace=s["space"])
    return s["c"]


def _cache(s):
    import telmo_amd

    if "cache" not in s:
        s["cache"] = telmo_amd.PagedCache(_context(), s["k"], s["v"], k_exps=s["k_exps"], v_exps=s["v_exps"])
    return s["cache"]


def _own_paged(s):
    import telmo_amd

    c = s["case"]
    if "attention" not in s:
        att = s["attention"] = telmo_amd.Attention(_context(), c["heads"], c["d"], kv_heads=c["kv_heads"], softcap=c["cap"],
                                                   left=None if c["left"] < 0 else c["left"], right=0, slopes=s.get("slopes"))
        s["space"] = _workspace(att.workspace_bytes(rows=s["q"].shape[0], keys=c["cached"], batch=c["sequences"]))
    s["attention"].paged(s["q"], _cache(s), s["tables"], s["lens"], s["out"], q_starts=s["starts"], longest=s["longest"],
                         prefix=s["prefix"], workspace=s["space"])
    return s["out"]


def _own_append(s):
    import telmo_amd

    c = s["case"]
    rotary = None
    if c["dim"]:
        rotary = _keep(("rotary", c["dim"], c["interleaved"]),
                       lambda: telmo_amd.Rotary(_context(), c["dim"], base=ROTARY_BASE, interleaved=c["interleaved"]))
    _cache(s).append(s["k_rows"], s["v_rows"], s["tables"], s["lens"], q_starts=s["starts"], longest=s["longest"], rotary=rotary)
    return [s["k"], s["v"], s["k_exps"], s["v_exps"]]


def _own_sample(s):
    import telmo_amd

    if "sampler" not in s:
        s["sampler"] = telmo_amd.Sampler(_context(), **s["options"])
        s["space"] = _workspace(s["sampler"].workspace_bytes(*s["logits"].shape))
    s["sampler"].sample(s["logits"], s["uniforms"], s["tokens"], s["probs"], workspace=s["space"])
    return [s["tokens"], s["probs"]]


OWN = {"product": _own_product, "paged": _own_paged, "append": _own_append, "sample": _own_sample}


def run(state):
    if own:
        return OWN[state["case"]["kind"]](state)
    return PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------- the work

def work(case):
    kind = case["kind"]
    if kind == "product":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * BYTES[case["type"]] + n * k + 4 * -(-n // GROUP) * -(-k // GROUP) + m * n * BYTES[case["to"]] +
                (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "sample":
        values = case["rows"] * case["n"]
        return {"bytes": values * BYTES[case["type"]] + 12 * case["rows"], "flops": 3 * values}
    shapes = _shapes(case, 1)
    rows, kv, d = sum(shapes["new"]), case["kv_heads"], case["d"]
    if kind == "append":
        blocks = sum((total - 1) // case["block"] - (total - new) // case["block"] + 1
                     for new, total in zip(shapes["new"], shapes["lens"]))
        return {"bytes": 2 * rows * kv * d * (BYTES[case["type"]] + 1) + 2 * blocks * kv, "flops": 3 * rows * kv * case["dim"]}
    left = case["left"] if case["left"] >= 0 else 1 << 40
    pairs, keys = 0, 0
    for new, total in zip(shapes["new"], shapes["lens"]):
        at = np.arange(total - new, total)
        first = np.maximum(at - left, 0)
        prefix = min(case["prefix"], total)
        pairs += int((at - first + 1 + np.minimum(first, prefix) + np.maximum(prefix - at - 1, 0)).sum())
        keys += int(total - first[0] + min(prefix, int(first[0])))
    return {"bytes": 2 * BYTES[case["type"]] * rows * case["heads"] * d + 2 * keys * kv * d + 2 * -(-keys // case["block"]) * kv,
            "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------- the outputs in 64 bits

def _nearest(x):
    """x (|x| <= 448, 64 bits) rounded to a multiple of its binade's eighth, or of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _fit(top):
    """The least whole e >= LOWEST with top <= 448 2^e, by trying."""
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 448.0))
    e = e + (top > 448.0 * torch.exp2(e)).double()
    return (e - (top <= 448.0 * torch.exp2(e - 1)).double()).clamp(min=LOWEST)


def _exact_product(case, s):
    m, k, n = case["m"], case["k"], case["n"]
    out = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    for a in range(0, k, GROUP):
        x = s["a"][:, a:a + GROUP].double()
        e = torch.exp2(_fit(x.abs().amax(1, keepdim=True)))
        x = _nearest(x / e) * e
        w = s["values"][:, a:a + GROUP].double()
        w = w * torch.repeat_interleave(s["scales"][:, a // GROUP].double(), GROUP)[:n, None]
        out.addmm_(x, w.t())
    if s["bias"] is not None:
        out += s["bias"].double()
    if case["act"] != "none":
        out = torch.relu(out) if case["act"] == "relu" else out * torch.sigmoid(out)
    return out * case["scale"]


def _exact_paged(case, s):
    group, d, page, block = case["heads"] // case["kv_heads"], case["d"], case["page"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for b, total in enumerate(s["lens"].tolist()):
        key = torch.arange(total, device="cuda")
        at, row = s["tables"][b].long()[key // page], key % page

        def of(name):
            x = s[name].view(torch.uint8)[at, row].view(E4M3).double()
            return x * torch.exp2(s[name + "_exps"][at, row // block].double())[..., None]

        k, v = of("k"), of("v")
        first, end = starts[b], starts[b + 1]
        position = torch.arange(total - (end - first), total, device="cuda")
        some = max(1, (1 << 25) // total)
        for h in range(case["heads"]):
            for x in range(first, end, some):
                rows = slice(x, min(x + some, end))
                distance = position[rows.start - first:rows.stop - first, None] - key
                score = s["q"][rows, h].double() @ k[:, h // group].t() / math.sqrt(d)
                if case["cap"]:
                    score = torch.tanh(score / case["cap"]) * case["cap"]
                if case["slopes"]:
                    score -= float(s["slopes"][h]) * distance.abs()
                hidden = distance < 0
                if case["left"] >= 0:
                    hidden = hidden | (distance > case["left"])
                score[hidden & (key >= case["prefix"])] = -math.inf
                out[rows, h] = torch.softmax(score, 1) @ v[:, h // group]
    return out


def _exact_append(case, s):
    page, block, dim = case["page"], case["block"], case["dim"]
    outs = [s[x].view(torch.uint8).clone().view(E4M3).double() for x in ("k", "v")]
    starts = s["starts"].tolist()
    for b, total in enumerate(s["lens"].tolist()):
        a, e = starts[b], starts[b + 1]
        position = torch.arange(total - (e - a), total, device="cuda")
        rows = [s["k_rows"][a:e].double(), s["v_rows"][a:e].double()]
        if dim:
            f = torch.from_numpy(np.power(ROTARY_BASE, -2 * np.arange(dim // 2) / dim)).cuda()
            turn = torch.polar(torch.ones((e - a, 1, dim // 2), dtype=torch.float64, device="cuda"),
                               torch.outer(position.double(), f)[:, None])
            first, second = (slice(0, dim, 2), slice(1, dim, 2)) if case["interleaved"] else (slice(0, dim // 2), slice(dim // 2, dim))
            z = torch.complex(rows[0][..., first], rows[0][..., second]) * turn
            rows[0][..., first], rows[0][..., second] = z.real.clone(), z.imag.clone()
        for x, (name, out) in enumerate(zip(("k", "v"), outs)):
            for n in range(int(position[0]) // block, (total - 1) // block + 1):
                lo, hi = max(n * block, int(position[0])), min((n + 1) * block, total)
                new = rows[x][lo - int(position[0]):hi - int(position[0])]
                p = int(s["tables"][b, n * block // page])
                r0, r = n * block % page, lo % page
                fit, had = _fit(new.abs().amax((0, 2))), s[name + "_exps"][p, r0 // block].double()
                if lo > n * block:
                    fit = torch.maximum(fit, had)
                    out[p, r0:r] = _nearest(out[p, r0:r] * torch.exp2(had - fit)[:, None])
                out[p, r:r + hi - lo] = _nearest(new * torch.exp2(-fit)[:, None])
    return outs + [None, None]


def _exact_sample(case, s):
    x, u = s["logits"].float().cpu().numpy().astype(np.float64), s["uniforms"].cpu().numpy().astype(np.float64)
    options = {}
    for name, value in s["options"].items():
        value = value.cpu().numpy() if isinstance(value, torch.Tensor) else np.full(case["rows"], value, np.float64)
        options[name] = value.astype(np.int64 if name == "top_k" else np.float32).astype(np.float64)
    probs = np.zeros(case["rows"])
    for r in range(case["rows"]):
        t, top_k = options["temperature"][r], int(options["top_k"][r])
        order = np.argsort(-x[r], kind="stable")
        if x[r, order[0]] == -np.inf:
            continue
        order = order[:1] if t == 0 else order[:top_k] if top_k else order
        w = np.exp((x[r, order] - x[r, order[0]]) / (t or 1.0))
        w = w[w > 0]
        if options["top_p"][r] < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w) - w, options["top_p"][r] * w.sum())))]
        w = w[:max(1, int((w >= options["min_p"][r]).sum()))]
        sums = np.cumsum(w)
        probs[r] = w[min(int(np.searchsorted(sums, u[r] * sums[-1], "right")), len(w) - 1)] / sums[-1]
    return [None, probs]


def exact(case, seed):
    s = prepare(case, seed)
    return {"product": _exact_product, "paged": _exact_paged, "append": _exact_append, "sample": _exact_sample}[case["kind"]](case, s)
