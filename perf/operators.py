"""The attention operators' work, as cases that can be timed and checked.

A case is a dict of plain values. ``listed()`` gives the standing ones and ``draw(rng)`` one more of the
same ranges; ``prepare(case, seed)`` makes what a program has in hand before the call, ``run(state)`` makes
one pass and returns its outputs (with ``own`` false by elementary torch operations in 32 bits, with ``own``
true by the framework's calls), ``exact(case, seed)`` gives the same outputs in 64 bits, and ``work(case)``
the bytes and operations that the pass cannot do without.

The kinds of case:

relative  the encoder layers' attention: f32 rows, q, k and v thirds of one product's rows, the scores of
          (q + u) k plus the position term (q + v) r of the distance (``Attention.forward``)
blocks    attention inside blocks of frames, one shared table of position rows (``Attention.forward``)
masked    attention over rows of packed sequences in 16 or 32 bits with capped scores, a bias by
          distance, a window, documents or a prefix, and shared key heads (``Attention.forward``)
paged     a chunk of new tokens, or a single one, of each sequence over its paged cache
          (``Attention.paged``)
rotary    rotary positions of rows, either layout, of part of the head or all of it, with frequencies
          scaled for long contexts (``Rotary.apply``)
append    new keys, rotated, and values into their pages (``PagedCache.append``)

Encoder sizes are the benchmark's: 8 heads of 128, 12.5 frames per second; blocks of 128 frames; the
others are generic. Rows are N(0, 1); scores are scaled by 1 / sqrt(d) throughout."""
import math

import numpy as np
import torch

own = False

HEADS, DIM, BLOCK = 8, 128, 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------ cases

def _masked(**kw):
    case = {"kind": "masked", "type": "bf16", "heads": 8, "kv_heads": 8, "d": 64, "lengths": "one", "rows": 1024,
            "sequences": 1, "cap": 0.0, "bias": "none", "left": -1, "right": -1, "prefix": 0, "documents": 0}
    case.update(kw)
    return case


def _paged(**kw):
    case = {"kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8, "d": 128, "sequences": 32, "new": 1,
            "ragged": True, "cached": 8192, "page": 16, "cap": 0.0, "left": -1, "bias": "none"}
    case.update(kw)
    return case


def listed():
    return [
        # One layer's attention over a minute of audio, the ordinary offline call.
        {"name": "relative, 60 s", "kind": "relative", "batch": 1, "rows": 750},
        # Batch transcription: sixteen such utterances stacked along the rows.
        {"name": "relative, 16 x 60 s", "kind": "relative", "batch": 16, "rows": 750},
        # The other encoder's: blocks of 128 frames, the last one short, one table for all heads.
        {"name": "blocks, 60 s", "kind": "blocks", "rows": 750},
        # A text encoder of 12 heads over texts packed one after another, a local layer of 64 tokens a side.
        dict(_masked(heads=12, kv_heads=12, rows=4096, documents=24, left=64, right=64), name="window, packed texts"),
        # Ragged sequences in half precision, prefix tokens seen by all, a slope for each head.
        dict(_masked(type="f16", heads=16, kv_heads=4, d=128, lengths="ragged", rows=5003, sequences=7, bias="slopes",
                     right=0, prefix=100), name="prefix and slopes, ragged"),
        # A long prompt of a causal decoder whose scores are capped.
        dict(_masked(heads=32, kv_heads=8, d=128, rows=8192, cap=50.0, right=0), name="capped, 8192 causal"),
        # Eight streams, one frame each over the frames before it: the smallest call.
        dict(_paged(type="f16", heads=8, kv_heads=8, sequences=8, cached=750, page=25), name="one token, 8 streams"),
        # A server's decode step over long caches.
        dict(_paged(), name="one token, 32 x 8192"),
        # A chunk of a long prompt over what is cached of it.
        dict(_paged(sequences=1, new=509, cached=32768, page=64, ragged=False), name="chunk of 509 over 32768"),
        # One row of each of eight streams: the smallest rotation.
        {"name": "rotary, 8 rows", "kind": "rotary", "type": "f32", "to": "f32", "rows": 8, "heads": 8, "d": 128,
         "dim": 128, "interleaved": False, "scaling": "none", "far": 4096},
        # The queries of a long prompt, half of each head rotated, far positions scaled by parts.
        {"name": "rotary, 16384 rows", "kind": "rotary", "type": "bf16", "to": "bf16", "rows": 16384, "heads": 32,
         "d": 128, "dim": 64, "interleaved": True, "scaling": "parts", "far": 131072},
        # Four prompts' f32 keys and values into 16-bit pages, each stopping inside a page.
        {"name": "append, 4 x 2047", "kind": "append", "type": "f32", "to": "bf16", "sequences": 4, "new": 2047,
         "kv_heads": 8, "d": 128, "dim": 128, "interleaved": False, "cached": 4096, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["relative", "relative", "blocks", "masked", "masked", "masked", "paged", "paged", "paged", "rotary",
                       "rotary", "append"])
    if kind == "relative":
        batch = rng.choice([1, 1, 2, 3, 8])
        return {"kind": kind, "batch": batch, "rows": _log(rng, 1, 2000 // batch)}
    if kind == "blocks":
        return {"kind": kind, "rows": _log(rng, 1, 6000)}
    if kind == "masked":
        kv = rng.choice([1, 2, 4, 5, 8])
        group = rng.choice([1, 1, 2, 3, 4, 7])
        sequences = rng.choice([1, 1, 2, 5, 9])
        rows = _log(rng, max(20, sequences), 4000)
        return _masked(type=rng.choice(["f16", "bf16", "bf16", "f32"]), heads=kv * group, kv_heads=kv,
                       d=rng.choice([32, 64, 64, 80, 128, 128, 192, 256]), lengths="ragged" if sequences > 1 else "one",
                       rows=rows, sequences=sequences, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                       bias=rng.choice(["none", "slopes", "table"]), left=rng.choice([-1, -1, 0, 17, 64, 300]),
                       right=rng.choice([-1, 0, 0, 64]), prefix=rng.choice([0, 0, 5, 70]),
                       documents=rng.choice([0, 0, 3, 11]))
    if kind == "paged":
        kv = rng.choice([1, 2, 4, 8])
        sequences = rng.choice([1, 1, 3, 8, 17])
        new = rng.choice([1, 1, 2, 5, _log(rng, 8, 300)])
        return _paged(type=rng.choice(["f16", "bf16", "f32"]), heads=kv * rng.choice([1, 2, 4, 6]), kv_heads=kv,
                      d=rng.choice([64, 96, 128, 128, 256]), sequences=sequences, new=new,
                      cached=_log(rng, new + 1, 24000 // sequences), page=rng.choice([1, 7, 16, 16, 64, 256]),
                      cap=rng.choice([0.0, 0.0, 40.0]), left=rng.choice([-1, -1, 200]), bias=rng.choice(["none", "slopes"]))
    if kind == "rotary":
        d = rng.choice([64, 80, 128, 256])
        kinds = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
        return {"kind": kind, "type": kinds[0], "to": kinds[1], "rows": _log(rng, 1, 12000), "heads": rng.choice([1, 3, 8, 16]),
                "d": d, "dim": rng.choice([d, d, d // 2, 16]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "base", "parts"]), "far": _log(rng, 1000, 2000000)}
    d = rng.choice([64, 128, 256])
    sequences = rng.choice([1, 3, 8, 20])
    new = _log(rng, 1, 4000 // sequences)
    return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "to": "bf16", "sequences": sequences, "new": new,
            "kv_heads": rng.choice([1, 2, 8]), "d": d, "dim": rng.choice([0, d, d // 2]), "interleaved": rng.random() < 0.5,
            "cached": new + _log(rng, 1, 4000), "page": rng.choice([1, 7, 16, 64])}


# ------------------------------------------------------------------------------- inputs from a seed

_stream = None


def _own_stream():
    """The program's one stream, torch's current stream from the first call on."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    torch.cuda.set_stream(_stream)


def _lengths(rng, total, parts):
    """`parts` lengths of any size, the empty one among them where there are many, whose sum is total."""
    cuts = np.sort(rng.integers(0, total + 1, parts - 1))
    return np.diff(np.concatenate([[0], cuts, [total]])).tolist()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return _ints([0] + np.cumsum(lengths).tolist())


def _shapes(case, seed):
    """The ragged sizes that the seed decides, on the host."""
    rng = np.random.default_rng([int(seed), 11])
    if case["kind"] == "blocks":
        rows = case["rows"]
        return {"lengths": [BLOCK] * (rows // BLOCK) + ([rows % BLOCK] if rows % BLOCK else [])}
    if case["kind"] == "masked":
        lengths = [case["rows"]] if case["lengths"] == "one" else _lengths(rng, case["rows"], case["sequences"])
        docs = None
        if case["documents"]:
            docs = np.concatenate([np.full(n, i) for i, n in enumerate(_lengths(rng, case["rows"], case["documents"]))])
        return {"lengths": lengths, "docs": docs, "prefix": [min(case["prefix"], n) for n in lengths]}
    if case["kind"] in ("paged", "append"):
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
    return {}


def prepare(case, seed):
    _own_stream()
    kind = case["kind"]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 29)

    def normal(*shape, type="f32"):
        return torch.randn(shape, generator=gen, device="cuda").to(TYPES[type])

    s = {"case": case}
    shapes = _shapes(case, seed)
    if kind in ("relative", "blocks"):
        rows = case["rows"] * case.get("batch", 1)
        qkv = normal(rows, 3 * HEADS * DIM)
        s["q"], s["k"], s["v"] = qkv.split(HEADS * DIM, dim=1)
        s["out"] = torch.empty((rows, HEADS * DIM), device="cuda")
    if kind == "relative":
        s["rel"] = normal(2 * case["rows"] - 1, HEADS * DIM)
        s["u"], s["w"] = 0.5 * normal(HEADS, DIM), 0.5 * normal(HEADS, DIM)
    elif kind == "blocks":
        s["rel"] = normal(2 * BLOCK - 1, DIM)
        s["starts"] = _starts(shapes["lengths"])
        s["longest"] = max(shapes["lengths"])
    elif kind == "masked":
        rows, heads, d = case["rows"], case["heads"], case["d"]
        s["q"] = normal(rows, heads, d, type=case["type"])
        s["k"], s["v"] = normal(rows, case["kv_heads"], d, type=case["type"]), normal(rows, case["kv_heads"], d, type=case["type"])
        s["out"] = torch.empty_like(s["q"])
        lengths = shapes["lengths"]
        s["starts"], s["longest"] = _starts(lengths), max(lengths)
        s["docs"] = None if shapes["docs"] is None else _ints(shapes["docs"])
        s["prefix"] = _ints(shapes["prefix"]) if case["prefix"] else None
    elif kind == "paged":
        heads, kv, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
        s["q"] = normal(sum(shapes["new"]), heads, d, type=case["type"])
        s["k"] = normal(shapes["pages"], page, kv, d, type=case["type"])
        s["v"] = normal(shapes["pages"], page, kv, d, type=case["type"])
        s["out"] = torch.empty_like(s["q"])
        s["starts"], s["longest"] = _starts(shapes["new"]), max(shapes["new"])
        s["lens"], s["tables"] = _ints(shapes["lens"]), _ints(shapes["tables"])
    elif kind == "rotary":
        s["x"] = normal(case["rows"], case["heads"], case["d"], type=case["type"])
        s["out"] = torch.empty((case["rows"], case["heads"], case["d"]), dtype=TYPES[case["to"]], device="cuda")
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=gen, device="cuda", dtype=torch.int32)
    elif kind == "append":
        kv, d, page = case["kv_heads"], case["d"], case["page"]
        rows = sum(shapes["new"])
        s["k_rows"], s["v_rows"] = normal(rows, kv, d, type=case["type"]), normal(rows, kv, d, type=case["type"])
        s["k"] = normal(shapes["pages"], page, kv, d, type=case["to"])
        s["v"] = normal(shapes["pages"], page, kv, d, type=case["to"])
        s["starts"], s["longest"] = _starts(shapes["new"]), max(shapes["new"])
        s["lens"], s["tables"] = _ints(shapes["lens"]), _ints(shapes["tables"])
    if case.get("bias", "none") == "slopes":
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"])
    elif case.get("bias", "none") == "table":
        s["table"] = normal(case["heads"], 2 * 40 + 1)  # distances past 40 share the last entry
    return s


# --------------------------------------------------------------------------------- the plain forms

def _attend(q, k, v, scale, shown, cap=0.0, bias=None, term=None):
    """softmax(cap tanh(scale (q k' + term) / cap) + bias) v over the keys that are shown, for q [..., n, d],
    k and v [..., m, d] in 32 bits; a row that is shown nothing gives zeros."""
    s = q @ k.transpose(-1, -2)
    if term is not None:
        s = s + term
    s = s * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if bias is not None:
        s = s + bias
    if shown is not None:
        s = s.masked_fill(~shown, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total == 0, torch.ones_like(total), total)


def _distance_bias(state, distance):
    """The bias [heads, ...] of the distances key - query."""
    if "slopes" in state:
        return -state["slopes"].view(-1, *[1] * distance.dim()) * distance.abs().float()
    if "table" in state:
        span = (state["table"].shape[1] - 1) // 2
        return state["table"][:, (distance.clamp(-span, span) + span).long()]
    return None


def _plain_relative(s):
    c = s["case"]
    batch, rows, distances = c["batch"], c["rows"], 2 * c["rows"] - 1
    q, k, v = (s[n].reshape(batch, rows, HEADS, DIM).transpose(1, 2) for n in ("q", "k", "v"))
    rel = s["rel"].view(distances, HEADS, DIM).transpose(0, 1)
    i = torch.arange(rows, device="cuda")
    at = (i[None, :] - i[:, None] + rows - 1).expand(batch, HEADS, rows, rows)
    term = torch.gather((q + s["w"][:, None]) @ rel.transpose(1, 2), 3, at)
    out = _attend(q + s["u"][:, None], k, v, DIM ** -0.5, None, term=term)
    return out.transpose(1, 2).reshape(batch * rows, HEADS * DIM)


def _plain_blocks(s):
    rows = s["case"]["rows"]
    blocks = -(-rows // BLOCK)
    pad = blocks * BLOCK - rows
    q, k, v = (torch.cat([s[n], torch.zeros(pad, HEADS * DIM, device="cuda")]).view(blocks, BLOCK, HEADS, DIM).transpose(1, 2)
               for n in ("q", "k", "v"))
    i = torch.arange(BLOCK, device="cuda")
    at = (i[None, :] - i[:, None] + BLOCK - 1).expand(blocks, HEADS, BLOCK, BLOCK)
    term = torch.gather(q @ s["rel"].t(), 3, at)
    real = (torch.arange(blocks * BLOCK, device="cuda") < rows).view(blocks, 1, 1, BLOCK)
    out = _attend(q, k, v, DIM ** -0.5, real, term=term)
    return out.transpose(1, 2).reshape(blocks * BLOCK, HEADS * DIM)[:rows]


def _shown(distance, left, right):
    """Which distances key - query lie in the window."""
    shown = torch.ones_like(distance, dtype=torch.bool)
    if left >= 0:
        shown = shown & (distance >= -left)
    if right >= 0:
        shown = shown & (distance <= right)
    return shown


def _plain_masked(s):
    c = s["case"]
    rows, heads, kv, d = c["rows"], c["heads"], c["kv_heads"], c["d"]
    q = s["q"].float().transpose(0, 1).reshape(kv, heads // kv, rows, d)
    k, v = s["k"].float().transpose(0, 1).unsqueeze(1), s["v"].float().transpose(0, 1).unsqueeze(1)
    i = torch.arange(rows, device="cuda")
    which = torch.searchsorted(s["starts"][1:].long(), i, right=True)
    distance = i[None, :] - i[:, None]
    shown = _shown(distance, c["left"], c["right"])
    if s["prefix"] is not None:
        shown = shown | ((i - s["starts"].long()[which]) < s["prefix"].long()[which])[None, :]
    shown = shown & (which[None, :] == which[:, None])
    if s["docs"] is not None:
        shown = shown & (s["docs"][None, :] == s["docs"][:, None])
    bias = _distance_bias(s, distance)
    if bias is not None:
        bias = bias.view(kv, heads // kv, rows, rows)
    out = _attend(q, k, v, d ** -0.5, shown, cap=c["cap"], bias=bias)
    return out.reshape(heads, rows, d).transpose(0, 1).to(s["q"].dtype)


def _plain_paged(s):
    c = s["case"]
    heads, kv, d, n, new = c["heads"], c["kv_heads"], c["d"], c["sequences"], s["longest"]
    tables, lens, starts = s["tables"].long(), s["lens"].long(), s["starts"].long()
    held = min(tables.shape[1] * c["page"], c["cached"])
    k, v = (s[x][tables].reshape(n, -1, kv, d)[:, :held].float().permute(0, 2, 1, 3).unsqueeze(2) for x in ("k", "v"))
    counts = starts[1:] - starts[:-1]
    r, j = torch.arange(new, device="cuda"), torch.arange(held, device="cuda")
    rows = (starts[:-1, None] + r).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].view(n, new, kv, heads // kv, d).permute(0, 2, 3, 1, 4)
    distance = j - (lens[:, None, None] - counts[:, None, None] + r[:, None])
    shown = (_shown(distance, c["left"], 0) & (j < lens[:, None, None]))[:, None, None]
    bias = _distance_bias(s, distance)
    if bias is not None:
        bias = bias.view(kv, heads // kv, n, new, held).permute(2, 0, 1, 3, 4)
    out = _attend(q, k, v, d ** -0.5, shown, cap=c["cap"], bias=bias)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, new, heads, d)
    return out[r < counts[:, None]].to(s["q"].dtype)


ROTARY_BASE, FACTOR, ORIGINAL, SLOW, FAST = 10000.0, 8.0, 4096, 1.0, 32.0


def _frequencies(case):
    """Radians per position of each pair, in 64 bits, and the amplitude of the rotated values."""
    dim, scaling = case["dim"], case.get("scaling", "none")
    i = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
    if scaling == "base":  # the slowest pair turns FACTOR times slower, the fastest as before
        return (ROTARY_BASE * FACTOR ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
    f = ROTARY_BASE ** (-2.0 * i / dim)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "parts":  # by the turns a pair makes in the original context
        keep = ((ORIGINAL * f / (2 * math.pi) - SLOW) / (FAST - SLOW)).clamp(0.0, 1.0)
        return f * keep + f / FACTOR * (1.0 - keep), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


def _rotate(x, positions, case):
    """x [rows, heads, d] in 32 bits, its first dim values rotated by positions [rows]."""
    dim = case["dim"]
    if not dim:
        return x
    f, amplitude = _frequencies(case)
    angle = positions.double()[:, None, None] * f  # 64 bits: a far position's angle has no place in 32
    cos, sin = (torch.cos(angle) * amplitude).float(), (torch.sin(angle) * amplitude).float()
    turned, rest = x[..., :dim], x[..., dim:]
    if case["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        pair = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        pair = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([pair, rest], -1)


def _plain_rotary(s):
    return _rotate(s["x"].float(), s["positions"], s["case"]).to(TYPES[s["case"]["to"]])


def _slots(s, page):
    """Each new row's position and its place among all pages' rows."""
    starts, lens = s["starts"].long(), s["lens"].long()
    row = torch.arange(s["k_rows"].shape[0], device="cuda")
    which = torch.searchsorted(starts[1:], row, right=True)
    position = lens[which] - starts[which + 1] + row
    return position, s["tables"].long()[which, position // page] * page + position % page


def _plain_append(s):
    c = s["case"]
    position, slot = _slots(s, c["page"])
    s["k"].flatten(0, 1)[slot] = _rotate(s["k_rows"].float(), position, c).to(s["k"].dtype)
    s["v"].flatten(0, 1)[slot] = s["v_rows"].to(s["v"].dtype)
    return [s["k"], s["v"]]


PLAIN = {"relative": _plain_relative, "blocks": _plain_blocks, "masked": _plain_masked, "paged": _plain_paged,
         "rotary": _plain_rotary, "append": _plain_append}


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


def _attention(s, heads, kv_heads, d, **options):
    import telmo_amd

    if "attention" not in s:
        bias = {n: s[n] for n in ("slopes", "table") if n in s}
        s["attention"] = telmo_amd.Attention(_context(), heads, d, kv_heads=kv_heads, **options, **bias)
    return s["attention"]


def _window(n):
    return None if n < 0 else n


def _workspace(att, **sizes):
    """One workspace for all calls on the program's stream, as large as the largest wants it."""
    want = att.workspace_bytes(**sizes)
    have = _kept.get("workspace")
    if have is None or have.numel() < want:
        have = _kept["workspace"] = torch.empty(max(want, 1 << 20), dtype=torch.uint8, device="cuda")
    return have


def _rotary(case):
    import telmo_amd

    keys = ("dim", "interleaved", "scaling")
    scaling = case.get("scaling", "none")
    options = {} if scaling == "none" else {"scaling": scaling, "factor": FACTOR}
    if scaling == "parts":
        options.update(original=ORIGINAL, slow=SLOW, fast=FAST)
    return _keep(("rotary",) + tuple(case.get(k) for k in keys),
                 lambda: telmo_amd.Rotary(_context(), case["dim"], base=ROTARY_BASE, interleaved=case["interleaved"], **options))


def _own_relative(s):
    c = s["case"]
    att = _attention(s, HEADS, HEADS, DIM)
    if "space" not in s:
        s["space"] = _workspace(att, rows=c["batch"] * c["rows"], keys=c["rows"], batch=c["batch"])
    att.forward(s["q"], s["k"], s["v"], s["out"], batch=c["batch"], rel=s["rel"], rel_u=s["u"], rel_v=s["w"],
                workspace=s["space"])
    return s["out"]


def _own_blocks(s):
    att = _attention(s, HEADS, HEADS, DIM)
    att.forward(s["q"], s["k"], s["v"], s["out"], q_starts=s["starts"], longest=s["longest"], rel=s["rel"])
    return s["out"]


def _own_masked(s):
    c = s["case"]
    att = _attention(s, c["heads"], c["kv_heads"], c["d"], softcap=c["cap"], left=_window(c["left"]), right=_window(c["right"]))
    if "space" not in s:
        s["space"] = _workspace(att, rows=c["rows"], keys=s["longest"], batch=len(s["starts"]) - 1)
    att.forward(s["q"], s["k"], s["v"], s["out"], q_starts=s["starts"], longest=s["longest"], prefix=s["prefix"],
                q_docs=s["docs"], workspace=s["space"])
    return s["out"]


def _cache(s):
    import telmo_amd

    if "cache" not in s:
        s["cache"] = telmo_amd.PagedCache(_context(), s["k"], s["v"])
    return s["cache"]


def _own_paged(s):
    c = s["case"]
    att = _attention(s, c["heads"], c["kv_heads"], c["d"], softcap=c["cap"], left=_window(c["left"]), right=0)
    if "space" not in s:
        s["space"] = _workspace(att, rows=s["q"].shape[0], keys=c["cached"], batch=c["sequences"])
    att.paged(s["q"], _cache(s), s["tables"], s["lens"], s["out"], q_starts=s["starts"], longest=s["longest"],
              workspace=s["space"])
    return s["out"]


def _own_rotary(s):
    _rotary(s["case"]).apply(s["x"], s["out"], s["positions"])
    return s["out"]


def _own_append(s):
    c = s["case"]
    _cache(s).append(s["k_rows"], s["v_rows"], s["tables"], s["lens"], q_starts=s["starts"], longest=s["longest"],
                     rotary=_rotary(c) if c["dim"] else None)
    return [s["k"], s["v"]]


OWN = {"relative": _own_relative, "blocks": _own_blocks, "masked": _own_masked, "paged": _own_paged,
       "rotary": _own_rotary, "append": _own_append}


def run(state):
    if own:
        return OWN[state["case"]["kind"]](state)
    return PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------- the work

def _pairs(case, seed=1):
    """Query-key pairs of one head that the masks leave, and the keys that some query sees."""
    shapes = _shapes(case, seed)
    kind = case["kind"]
    if kind == "relative":
        return case["batch"] * case["rows"] ** 2, case["batch"] * case["rows"]
    if kind == "blocks":
        return sum(n * n for n in shapes["lengths"]), case["rows"]
    pairs, keys = 0, 0
    left = case["left"] if case["left"] >= 0 else 1 << 40
    if kind == "paged":
        for new, total in zip(shapes["new"], shapes["lens"]):
            at = np.arange(total - new, total)
            pairs += int((at - np.maximum(at - left, 0) + 1).sum())
            keys += int(total - max(0, total - new - left))
        return pairs, keys
    right = case["right"] if case["right"] >= 0 else 1 << 40
    at = 0
    for n, prefix in zip(shapes["lengths"], shapes["prefix"]):
        docs = shapes["docs"][at:at + n] if shapes["docs"] is not None else np.zeros(n, np.int64)
        at += n
        i = np.arange(n)
        first = np.searchsorted(docs, docs, "left") if n else i  # a document's rows follow one another
        last = np.searchsorted(docs, docs, "right") if n else i
        lo, hi = np.maximum(first, i - left), np.minimum(last, i + right + 1)
        before = np.clip(np.minimum(lo, np.minimum(prefix, last)) - first, 0, None)  # prefix keys outside the window
        after = np.clip(np.minimum(prefix, last) - np.maximum(hi, first), 0, None)
        pairs += int((np.maximum(hi - lo, 0) + before + after).sum())
        keys += n
    return pairs, keys


def work(case):
    kind = case["kind"]
    if kind in ("rotary", "append"):
        if kind == "rotary":
            values = case["rows"] * case["heads"] * case["d"]
            return {"bytes": values * (BYTES[case["type"]] + BYTES[case["to"]]) + 4 * case["rows"],
                    "flops": 3 * case["rows"] * case["heads"] * case["dim"]}
        rows = sum(_shapes(case, 1)["new"])
        values = 2 * rows * case["kv_heads"] * case["d"]
        return {"bytes": values * (BYTES[case["type"]] + BYTES[case["to"]]), "flops": 3 * rows * case["kv_heads"] * case["dim"]}
    pairs, keys = _pairs(case)
    if kind in ("relative", "blocks"):
        rows = case["rows"] * case.get("batch", 1)
        positions = (2 * case["rows"] - 1) * HEADS * DIM if kind == "relative" else (2 * BLOCK - 1) * DIM
        return {"bytes": 4 * (4 * rows * HEADS * DIM + positions), "flops": 6 * pairs * HEADS * DIM}
    rows = case["rows"] if kind == "masked" else sum(_shapes(case, 1)["new"])
    size = BYTES[case["type"]] * case["d"]
    return {"bytes": size * (2 * rows * case["heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * pairs * case["heads"] * case["d"]}


# ------------------------------------------------------------------------- the outputs in 64 bits

def _exact_rows(q, k, v, position, scale, see, cap=0.0, bias=None, rel=None, u=0.0, w=0.0):
    """One head's outputs by the definition, some queries at a time: q [n, d] at the key positions
    `position`, k and v [m, d]; see(rows, distance) tells which keys a query sees, bias(distance) the
    head's bias, rel(distance) the position rows' indices and the rows."""
    q, k, v = q.double(), k.double(), v.double()
    key = torch.arange(k.shape[0], device="cuda")
    out = torch.zeros_like(q)
    some = max(1, (1 << 25) // max(1, k.shape[0]))
    for a in range(0, q.shape[0], some):
        at = slice(a, min(a + some, q.shape[0]))
        distance = key[None, :] - position[at, None]
        score = (q[at] + u) @ k.t()
        if rel is not None:
            index, rows = rel
            score += ((q[at] + w) @ rows.double().t()).gather(1, index(distance))
        score *= scale
        if cap:
            score = torch.tanh(score / cap) * cap
        if bias is not None:
            score += bias(distance)
        score[~see(torch.arange(at.start, at.stop, device="cuda"), distance)] = -math.inf
        some_key = (score > -math.inf).any(1)
        weight = torch.softmax(score[some_key], 1)
        out[at][some_key] = weight @ v
    return out


def _exact_attention(case, s):
    kind = case["kind"]
    everything = lambda rows, distance: torch.ones_like(distance, dtype=torch.bool)  # noqa: E731
    if kind in ("relative", "blocks"):
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        if kind == "relative":
            edges = [(b * case["rows"], (b + 1) * case["rows"]) for b in range(case["batch"])]
            middle = case["rows"] - 1
        else:
            edges = [(a, min(a + BLOCK, case["rows"])) for a in range(0, case["rows"], BLOCK)]
            middle = BLOCK - 1
        for h in range(HEADS):
            col = slice(h * DIM, (h + 1) * DIM)
            rows = s["rel"][:, col] if kind == "relative" else s["rel"]
            u, w = (s["u"][h].double(), s["w"][h].double()) if kind == "relative" else (0.0, 0.0)
            for a, b in edges:
                out[a:b, col] = _exact_rows(s["q"][a:b, col], s["k"][a:b, col], s["v"][a:b, col],
                                            torch.arange(b - a, device="cuda"), 1.0 / math.sqrt(DIM), everything,
                                            rel=(lambda distance: distance + middle, rows), u=u, w=w)
        return out
    heads, group, d = case["heads"], case["heads"] // case["kv_heads"], case["d"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    left, right = case["left"], case.get("right", 0)

    def in_window(distance):
        ok = torch.ones_like(distance, dtype=torch.bool)
        if left >= 0:
            ok &= -distance <= left
        if right >= 0:
            ok &= distance <= right
        return ok

    starts = s["starts"].tolist()
    for b in range(len(starts) - 1):
        first, end = starts[b], starts[b + 1]
        if first == end:
            continue
        if kind == "masked":
            k, v, total = s["k"][first:end], s["v"][first:end], end - first
            prefix = int(s["prefix"][b]) if s["prefix"] is not None else 0
            docs = s["docs"][first:end] if s["docs"] is not None else None
        else:
            total = int(s["lens"][b])
            page = case["page"]
            held = s["tables"][b, :-(-total // page)].long()
            k, v = s["k"][held].flatten(0, 1)[:total], s["v"][held].flatten(0, 1)[:total]
            prefix, docs = 0, None
        position = torch.arange(total - (end - first), total, device="cuda")
        key = torch.arange(total, device="cuda")

        def see(rows, distance):
            ok = in_window(distance) | (key < prefix)
            return ok if docs is None else ok & (docs[rows][:, None] == docs[None, :])

        for h in range(heads):
            bias = None
            if "slopes" in s:
                bias = lambda distance: -float(s["slopes"][h]) * distance.abs()  # noqa: E731
            elif "table" in s:
                span = s["table"].shape[1] // 2
                bias = lambda distance: s["table"][h].double()[distance.clamp(-span, span) + span]  # noqa: E731
            out[first:end, h] = _exact_rows(s["q"][first:end, h], k[:, h // group], v[:, h // group], position,
                                            1.0 / math.sqrt(d), see, cap=case["cap"], bias=bias)
    return out


def _exact_turn(x, positions, case):
    """The pairs of x [rows, heads, d] as complex numbers times amplitude e^(i angle)."""
    x, dim = x.double().clone(), case["dim"]
    if not dim:
        return x
    i = np.arange(dim // 2, dtype=np.float64)
    f, amplitude, scaling = ROTARY_BASE ** (-2 * i / dim), 1.0, case.get("scaling", "none")
    if scaling == "linear":
        f = f / FACTOR
    elif scaling == "base":
        f = np.power(ROTARY_BASE * np.power(FACTOR, dim / (dim - 2)), -2 * i / dim)
    elif scaling == "parts":
        turns = ORIGINAL * f / (2 * np.pi)
        keep = np.clip((turns - SLOW) / (FAST - SLOW), 0, 1)
        f, amplitude = keep * f + (1 - keep) * f / FACTOR, 0.1 * math.log(FACTOR) + 1
    angle = torch.outer(positions.double(), torch.from_numpy(f).cuda())
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    first, second = (slice(0, dim, 2), slice(1, dim, 2)) if case["interleaved"] else (slice(0, dim // 2), slice(dim // 2, dim))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_turn(s["x"], s["positions"], case)
    if case["kind"] == "append":
        k, v, page = s["k"].double(), s["v"].double(), case["page"]
        starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].long()
        for b, total in enumerate(lens):
            a, e = starts[b], starts[b + 1]
            position = torch.arange(total - (e - a), total, device="cuda")
            at = (tables[b][position // page], position % page)
            k[at] = _exact_turn(s["k_rows"][a:e], position, case)
            v[at] = s["v_rows"][a:e].double()
        return [k, v]
    return _exact_attention(case, s)
