"""The attention operators as programs run them, on an MI355X: the attention argument of the Conformer layer
and the Granite block, and a token-by-token pass (rotate, append, attend over the cache)."""
import math

import numpy as np
import pytest

import bench
from attention_oracle import attend, rotate, shown_pairs, tolerance
from test_gpu_attention import check, dtype, floats, ints, position_rows, say
from test_gpu_layer import FF, K, close, device_layer

pytestmark = pytest.mark.gpu

D, HEADS, DIM, BLOCK = 1024, 8, 128, 128


def check_rows(got, q, k, v, rel, u, w):
    """One sequence's [n, D] outputs of all heads against the definition."""
    n = q.shape[0]
    for h in range(HEADS):
        col = slice(h * DIM, (h + 1) * DIM)
        uh, wh = (None if x is None else x[h].astype(np.float64) for x in (u, w))
        want, size = attend(q[:, col], k[:, col], v[:, col], DIM**-0.5, np.ones((n, n), bool),
                            rel=position_rows(n, n, h, rel, DIM), u=uh, w=wh)
        check(got[:, col], want, tolerance("f32", DIM, n, size, np.abs(v[:, col]).max(), True))


def test_conformer_layer_with_relative_positions(tk):
    """Two stacked utterances: the layer hands its qkv rows and projected positions to the attention, takes
    its rows, and otherwise runs as with any other attention that returns those rows."""
    import torch

    import telmo_amd
    from telmo_amd.conformer import ConformerLayer

    t, utterances = 150, 2
    frames = t // utterances
    mats, norms, dw_w, dw_b = bench.layer_params(1700)
    pv, ps = bench.panel_layout(bench.synth_int8(D, D, 1750), bench.synth_scales(D, 1751))
    weights = device_layer(tk, dict(mats, pos=(pv, ps, D, D)), norms, dw_w, dw_b)
    x = bench.synth_normal((t, D), 18)
    pos = floats(bench.synth_normal((2 * frames - 1, D), 19))
    u, w = 0.3 * bench.synth_normal((HEADS, DIM), 20), 0.3 * bench.synth_normal((HEADS, DIM), 21)
    layer, att = ConformerLayer(tk, D, FF, K, t), telmo_amd.Attention(tk, HEADS, DIM)
    space = torch.empty(att.workspace_bytes(t, frames, utterances) + 16, dtype=torch.uint8, device="cuda")
    out, p_out = (torch.zeros((n, D), device="cuda") for n in (t, 2 * frames - 1))
    run = att.for_layer(out, batch=utterances, rel_u=floats(u), rel_v=floats(w), workspace=space)
    seen = {}

    def attention(qkv, positions):
        seen["qkv"] = qkv.clone()
        return run(qkv, positions)

    say("conformer layer", t)
    xd = torch.from_numpy(x.copy()).cuda()
    layer.forward(xd, t, weights, utterances=utterances, attention=attention, pos=pos, p_out=p_out)
    tk.synchronize()
    qkv, rel, got = seen["qkv"].double().cpu().numpy(), p_out.cpu().numpy(), out.double().cpu().numpy()
    for a in range(0, t, frames):
        q, k, v = (qkv[a:a + frames, i * D:(i + 1) * D] for i in range(3))
        check_rows(got[a:a + frames], q, k, v, rel, u, w)
    again = torch.from_numpy(x.copy()).cuda()
    layer.forward(again, t, weights, utterances=utterances, attention=lambda qkv, p: out.clone(), pos=pos, p_out=p_out)
    tk.synchronize()
    assert torch.equal(again, xd)
    close([weights])


def test_granite_block_with_blocks_of_frames(tk):
    import torch

    import telmo_amd
    from telmo_amd.granite import GraniteBlock

    t = 2 * BLOCK + 37
    params = bench.granite_block_params(1800, False)
    weights = bench.upload_granite_block(tk, params)
    block = GraniteBlock(tk, D, bench.G_FF, bench.G_CC, bench.G_KERNEL, t)
    att, out = telmo_amd.Attention(tk, HEADS, DIM), torch.zeros((t, D), device="cuda")
    rel = bench.synth_normal((2 * BLOCK - 1, DIM), 22)
    edges = [0, BLOCK, 2 * BLOCK, t]
    run = att.for_layer(out, rel=floats(rel), q_starts=ints(edges), longest=BLOCK)
    seen = {}

    def attention(qkv):
        seen["qkv"] = qkv.clone()
        return run(qkv)

    say("granite block", t)
    xd = torch.from_numpy(bench.synth_normal((t, D), 23)).cuda()
    block.forward(xd, t, weights, attention=attention)
    tk.synchronize()
    qkv, got = seen["qkv"].double().cpu().numpy(), out.double().cpu().numpy()
    assert bool(torch.isfinite(xd).all())
    for a, b in zip(edges, edges[1:]):
        q, k, v = (qkv[a:b, i * D:(i + 1) * D] for i in range(3))
        check_rows(got[a:b], q, k, v, rel, None, None)
    close([weights])


@pytest.mark.parametrize("type,page", (("f32", 16), ("bf16", 7), ("f16", 64)))
def test_a_prompt_in_chunks_then_token_by_token(tk, gpu_stream, type, page):
    """Two sequences, each fed in chunks and then by single tokens replayed from one captured graph, against
    the causal attention of the whole sequence."""
    import torch

    import telmo_amd

    heads, kv, d, dim = 4, 2, 64, 32
    totals, chunks = (90, 77), ((50, 41), (30, 30), (1, 1), (1, 1), (1, 1), (1, 1))
    rng = np.random.default_rng(12)
    values = [rng.standard_normal((2, max(totals), n, d)).astype(np.float32) for n in (heads, kv, kv)]
    rows = [torch.from_numpy(x).to(dtype(type)) for x in values]
    exact = [x.double().numpy() for x in rows]
    width = -(-max(totals) // page)
    tables = ints(rng.permutation(2 * width).reshape(2, width))
    store = [torch.full((2 * width, page, kv, d), float("nan"), dtype=dtype(type), device="cuda") for _ in "kv"]
    cache, rotary = telmo_amd.PagedCache(tk, *store), telmo_amd.Rotary(tk, dim, scaling="linear", factor=2.0)
    att = telmo_amd.Attention(tk, heads, d, kv_heads=kv, right=0)
    space = torch.empty(att.workspace_bytes(200, max(totals), 2) + 16, dtype=torch.uint8, device="cuda")
    lens = ints([0, 0])
    f, amplitude = telmo_amd.rotary_frequencies(dim, scaling="linear", factor=2.0)
    outs = [[], []]
    done, graph, bufs = [0, 0], None, None

    def step(q, k, v, positions, turned, out, starts):
        rotary.apply(q, turned, positions)
        cache.append(k, v, tables, lens, q_starts=starts, rotary=rotary)
        att.paged(turned, cache, tables, lens, out, q_starts=starts, workspace=space)

    for new in chunks:
        say("chunk", type, new, done)
        q, k, v = (torch.cat([x[b, done[b]:done[b] + new[b]] for b in (0, 1)]).cuda() for x in rows)
        at = ints(np.concatenate([np.arange(done[b], done[b] + new[b]) for b in (0, 1)]))
        lens.copy_(ints([done[b] + new[b] for b in (0, 1)]))
        if new == (1, 1):
            if graph is None:
                bufs = [q, k, v, at, torch.zeros_like(q), torch.zeros_like(q), ints([0, 1, 2])]
                step(*bufs)
                tk.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=gpu_stream):
                    step(*bufs)
            else:
                for into, x in zip(bufs, (q, k, v, at)):
                    into.copy_(x)
                bufs[5].fill_(3.0)
                graph.replay()
            out = bufs[5].clone()
        else:
            out = torch.zeros_like(q)
            step(q, k, v, at, torch.zeros_like(q), out, ints([0, new[0], sum(new)]))
        tk.synchronize()
        got = out.double().cpu().numpy()
        outs[0].append(got[:new[0]])
        outs[1].append(got[new[0]:])
        done = [done[b] + new[b] for b in (0, 1)]
    for b in (0, 1):
        n = done[b]
        got = np.concatenate(outs[b])
        q, k = (rotate(x[b, :n], np.arange(n), f, amplitude, dim, False) for x in exact[:2])
        v = exact[2][b, :n]
        # Rotated values are off by up to half a step of their type and of what sine and cosine keep.
        each = {"f32": 2.0**-20, "f16": 2.0**-11 + 2.0**-20, "bf16": 2.0**-8}[type]
        turn = d**-0.5 * sum(np.abs(q).max() * np.abs(k).max() * d * e for e in (each, each))
        for h in range(heads):
            g = h // (heads // kv)
            want, size = attend(q[:, h], k[:, g], v[:, g], d**-0.5, shown_pairs(n, n, None, 0))
            top = np.abs(v).max()
            check(got[:, h], want, tolerance(type, d, n, size, top, False) + 2 * top * math.expm1(turn))
