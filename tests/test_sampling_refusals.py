"""Drawing tokens without a GPU: what it refuses, through the C ABI (a call whose arguments stand answers that the
context is null)."""
import pytest

OK, NULL, SHAPE, ALIGN, UNSUPPORTED, ARG = -1, -1, -2, -3, -5, -7  # OK: only the context is missing
AT = 1 << 20
NAN, INF = float("nan"), float("inf")


def call(type=0, logits=AT, logits_len=None, ld=40000, rows=5, n=40000, uniforms=AT * 16, uniforms_len=5, tokens=AT * 17, tokens_len=5,
         probs=AT * 18, probs_len=5, space=AT * 32, space_len=None, options=True, **fields):
    from telmo_amd import _lib

    L = _lib.lib()
    o = _lib.Sampling(1.0, 0, 1.0, 0.0)
    for name, value in fields.items():
        setattr(o, name, value)
    need = L.tg_sample_workspace_bytes(rows, n) if space_len is None else space_len
    return L.tg_sample_device(None, type, logits, (rows - 1) * ld + n if logits_len is None else logits_len, ld, rows, n,
                              o if options else None, uniforms, uniforms_len, tokens, tokens_len, probs, probs_len, space, need)


@pytest.mark.parametrize("kw,code", [
    ({}, OK), (dict(options=False), NULL), (dict(type=3), ARG), (dict(type=4), ARG), (dict(temperature=-1.0), ARG), (dict(temperature=NAN), ARG),
    (dict(temperature=INF), ARG), (dict(temperature=0.0), OK), (dict(top_k=-1), ARG), (dict(top_k=7), OK), (dict(top_p=1.1), ARG),
    (dict(top_p=NAN), ARG), (dict(top_p=-0.1), ARG), (dict(top_p=0.0), OK), (dict(min_p=1.1), ARG), (dict(min_p=NAN), ARG), (dict(min_p=1.0), OK),
    (dict(rows=(1 << 20) + 1, logits_len=1 << 60), UNSUPPORTED), (dict(n=(1 << 22) + 1, ld=1 << 23), UNSUPPORTED), (dict(ld=39999), SHAPE),
    (dict(logits_len=4 * 40000 + 39999), SHAPE), (dict(uniforms_len=4), SHAPE), (dict(tokens_len=4), SHAPE), (dict(probs_len=4), SHAPE),
    (dict(probs=None, probs_len=0), OK), (dict(logits=None), NULL), (dict(uniforms=None), NULL), (dict(tokens=None), NULL),
    (dict(n=0, ld=0, logits=None, space=None), OK), (dict(logits=AT + 2), ALIGN), (dict(logits=AT + 2, type=1), OK), (dict(tokens=AT * 17 + 2), ALIGN),
    (dict(probs=AT * 18 + 1), ALIGN), (dict(space=None), SHAPE), (dict(space_len=100), SHAPE), (dict(space=AT * 32 + 8), ALIGN),
    (dict(temperatures=AT * 20, temperatures_len=4), SHAPE), (dict(temperatures=AT * 20, temperatures_len=5), OK),
    (dict(top_ks=AT * 20, top_ks_len=4), SHAPE), (dict(top_ps=AT * 20, top_ps_len=4), SHAPE), (dict(min_ps=AT * 20, min_ps_len=4), SHAPE),
    (dict(tokens=AT + 400), ARG), (dict(probs=AT * 16 + 16), ARG), (dict(probs=AT * 17 + 16), ARG), (dict(space=AT + 16), ARG),
    (dict(tokens=AT * 32 + 64), ARG), (dict(top_ks=AT * 17, top_ks_len=5), ARG), (dict(ld=1 << 61, logits_len=(1 << 64) - 1), SHAPE),
    (dict(n=32768, ld=32768, space=None), OK), (dict(n=32769, ld=32769, space=None), SHAPE),
])
def test_refusals(kw, code):
    assert call(**kw) == code


def test_workspaces():
    from telmo_amd import _lib

    f = _lib.lib().tg_sample_workspace_bytes
    assert f(5, 32768) == 0 and f(0, 50000) == 0
    assert f(3, 50000) == 3 * f(1, 50000) > 0 and f(1, 131072) > f(1, 50000)
    assert f(1, (1 << 22) + 1) == f((1 << 20) + 1, 50000) == 0
