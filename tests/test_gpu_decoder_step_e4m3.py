"""A decoder's steps in eight bits on an MI355X: products, the cache's appends and attention, and a token's drawing in one
run, prompts first and then single tokens from a captured graph that feeds each token to the next step."""
import numpy as np
import pytest

from attention_oracle import HALF_STEP, attend, rotate, shown_pairs
from e4m3_oracle import VALUES, half_step
from test_gpu_attention import check, ints, say
from test_gpu_cache_e4m3 import allowed
from test_gpu_e4m3_product import rounded_rows, stood_for
from test_gpu_sampling import draw

pytestmark = pytest.mark.gpu

HEADS, KV, D, WIDTH, VOCABULARY, PAGE, BLOCK, KEYS = 4, 2, 64, 256, 1000, 32, 16, 96
PROMPTS, STEPS = (40, 7, 1), 5
DRAWN = dict(temperature=0.9, top_k=60, top_p=0.95, min_p=0.01)


def host(t):
    return t.double().cpu().numpy()


class Decoder:
    def __init__(self, tk, seed):
        import torch

        import telmo_amd

        rng = np.random.default_rng(seed)
        self.tk, self.torch = tk, torch
        self.w, self.w64 = {}, {}
        for name, k, n in (("qkv", WIDTH, (HEADS + 2 * KV) * D), ("out", HEADS * D, WIDTH), ("logits", WIDTH, VOCABULARY)):
            codes, scales = telmo_amd.encode_e4m3(rng.standard_normal((n, k)) * (3.0 if name == "logits" else 1.0) / k**0.5, n, k)
            self.w[name] = telmo_amd.E4m3Weights.from_parts(tk, codes, scales)
            self.w64[name] = stood_for(codes, scales)
        self.embedding = torch.from_numpy(rng.standard_normal((VOCABULARY, WIDTH)).astype(np.float32)).cuda().bfloat16()
        batch, pages = len(PROMPTS), KEYS // PAGE
        self.tables = rng.permutation(batch * pages).reshape(batch, pages)
        self.codes = [torch.full((batch * pages, PAGE, KV, D), 0x7F, dtype=torch.uint8, device="cuda") for _ in "kv"]
        self.exps = [torch.full((batch * pages, PAGE // BLOCK, KV), 127, dtype=torch.int8, device="cuda") for _ in "kv"]
        self.cache = telmo_amd.PagedCache(tk, *self.codes, k_exps=self.exps[0], v_exps=self.exps[1])
        self.rotary = telmo_amd.Rotary(tk, D)
        self.attention = telmo_amd.Attention(tk, HEADS, D, kv_heads=KV, right=0)
        self.sampler = telmo_amd.Sampler(tk, **DRAWN)
        self.table, self.lengths = ints(self.tables), ints([0] * batch)

    def buffers(self, rows, starts):
        """What a step of so many rows reads and leaves."""
        torch, batch = self.torch, len(PROMPTS)
        new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device="cuda")
        space = max(self.attention.workspace_bytes(rows, KEYS, batch), *(w.workspace_bytes(rows) for w in self.w.values()),
                    self.sampler.workspace_bytes(batch, VOCABULARY))
        return dict(tokens=new(rows, dtype=torch.int32), positions=new(rows, dtype=torch.int32), starts=ints(starts),
                    last=ints(np.asarray(starts[1:]) - 1), x=new(rows, WIDTH), qkv=new(rows, (HEADS + 2 * KV) * D), q=new(rows, HEADS, D),
                    heads=new(rows, HEADS * D), y=new(rows, WIDTH), z=new(batch, WIDTH), logits=new(batch, VOCABULARY, dtype=torch.float32),
                    uniforms=new(batch, dtype=torch.float32), drawn=new(batch, dtype=torch.int32),
                    probs=new(batch, dtype=torch.float32), space=torch.zeros(space, dtype=torch.uint8, device="cuda"))

    def step(self, b):
        torch, tk = self.torch, self.tk
        rows = b["x"].shape[0]
        torch.index_select(self.embedding, 0, b["tokens"], out=b["x"])
        tk.linear_e4m3_device(b["x"], self.w["qkv"], b["qkv"], workspace=b["space"])
        q, k, v = (t.view(rows, -1, D) for t in b["qkv"].split((HEADS * D, KV * D, KV * D), 1))
        self.rotary.apply(q, b["q"], b["positions"])
        self.cache.append(k, v, self.table, self.lengths, q_starts=b["starts"], rotary=self.rotary)
        self.attention.paged(b["q"], self.cache, self.table, self.lengths, b["heads"].view(rows, HEADS, D), q_starts=b["starts"],
                             workspace=b["space"])
        tk.linear_e4m3_device(b["heads"], self.w["out"], b["y"], workspace=b["space"])
        torch.index_select(b["y"], 0, b["last"], out=b["z"])
        tk.linear_e4m3_device(b["z"], self.w["logits"], b["logits"], workspace=b["space"])
        self.sampler.sample(b["logits"], b["uniforms"], b["drawn"], b["probs"], workspace=b["space"])

    def held(self):
        """The keys and values that the cache stands for, in each sequence's order."""
        at = lambda x: x.cpu().numpy()[self.tables]
        return [(VALUES[at(c)] * 2.0 ** np.repeat(at(e).astype(np.float64), BLOCK, 2)[..., None]).reshape(len(PROMPTS), KEYS, KV, D)
                for c, e in zip(self.codes, self.exps)]

    def product(self, name, a, c):
        a, w = rounded_rows(host(a)), self.w64[name]
        want, sums = a @ w.T, np.abs(a) @ np.abs(w).T
        tol = (2 * a.shape[1] + 64) * HALF_STEP["f32"] * sums
        if c.dtype != self.torch.float32:
            for x in range(0, a.shape[1], 128):  # products in e4m3 that are aligned first
                tol = tol + 2.0**-10 * np.abs(a[:, x:x + 128]).max(1)[:, None] * np.abs(w[:, x:x + 128]).max(1)
            tol = tol + HALF_STEP["bf16"] * (np.abs(want) + tol)
        assert np.all(np.abs(host(c) - want) <= tol + 2.0**-120), name

    def check(self, b, new, lengths):
        """Each operator's results against its definition over what it was given."""
        import telmo_amd

        self.product("qkv", b["x"], b["qkv"])
        self.product("out", b["heads"], b["y"])
        self.product("logits", b["z"], b["logits"])
        _, k, v = (t.reshape(len(b["qkv"]), -1, D) for t in np.split(host(b["qkv"]), (HEADS * D, (HEADS + KV) * D), 1))
        got, q64, (ks, vs) = host(b["heads"]).reshape(-1, HEADS, D), host(b["q"]), self.held()
        f, amplitude = telmo_amd.rotary_frequencies(D)
        r = 0
        for s, (n, m) in enumerate(zip(new, lengths)):
            for x, stands, turned, exps in ((k, ks, True, self.exps[0]), (v, vs, False, self.exps[1])):
                at = np.arange(m - n, m)
                want = rotate(x[r:r + n], at, f, amplitude, D, False) if turned else x[r:r + n]
                e = exps.cpu().numpy()[self.tables[s]].reshape(-1, KV)[at // BLOCK].astype(np.float64)[..., None]
                slack = 2.0**-20 * np.abs(want).max()
                assert np.all(np.abs(stands[s, at] - want) <= half_step(np.abs(want) + slack, e) + slack)
            for h in range(HEADS):
                g = h // (HEADS // KV)
                want, size = attend(q64[r:r + n, h], ks[s, :m, g], vs[s, :m, g], D**-0.5, shown_pairs(n, m, None, 0))
                check(got[r:r + n, h], want, allowed("bf16", D, m, size, np.abs(vs[s, :m, g]).max()))
            r += n
        logits, u, tokens, probs = (x.cpu().numpy() for x in (b["logits"], b["uniforms"], b["drawn"], b["probs"]))
        for s in range(len(new)):
            token, prob, near = draw(logits[s], u[s], **DRAWN)
            assert near <= VOCABULARY * 2.0**-42 or tokens[s] == token
            assert abs(probs[s] - prob) <= 2.0**-23 * prob


def run(tk, gpu_stream, captured):
    import torch

    d, batch = Decoder(tk, 5), len(PROMPTS)
    rng = np.random.default_rng(6)
    starts = np.concatenate([[0], np.cumsum(PROMPTS)])
    b = d.buffers(sum(PROMPTS), starts)
    b["tokens"].copy_(ints(rng.integers(0, VOCABULARY, sum(PROMPTS))))
    b["positions"].copy_(ints(np.concatenate([np.arange(n) for n in PROMPTS])))
    b["uniforms"].copy_(torch.from_numpy(rng.random(batch).astype(np.float32)))
    d.lengths.copy_(ints(PROMPTS))
    d.step(b)
    torch.cuda.synchronize()
    d.check(b, PROMPTS, PROMPTS)
    tokens, one = [b["drawn"].tolist()], d.buffers(batch, list(range(batch + 1)))
    one["drawn"].copy_(b["drawn"])

    def next_step():
        one["tokens"].copy_(one["drawn"])
        one["positions"].copy_(d.lengths)
        d.lengths.add_(1)
        d.step(one)

    graph = None
    for i in range(STEPS):
        one["uniforms"].copy_(torch.from_numpy(rng.random(batch).astype(np.float32)))
        torch.cuda.synchronize()
        if captured and graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=gpu_stream):
                next_step()
        if captured:
            graph.replay()
        else:
            next_step()
        torch.cuda.synchronize()
        say("step", i, captured)
        lengths = [n + i + 1 for n in PROMPTS]
        assert d.lengths.tolist() == lengths
        d.check(one, (1,) * batch, lengths)
        tokens.append(one["drawn"].tolist())
    return tokens


def test_prompts_and_steps(tk, gpu_stream):
    """The captured run draws the eager one's tokens."""
    assert run(tk, gpu_stream, True) == run(tk, gpu_stream, False)
