"""What the eight-bit product and cache refuse with a GPU at hand: nothing is queued, and what they were to write is left
as it was."""
import pytest

pytestmark = pytest.mark.gpu

ALIGN, ARG, NULL, SHAPE, UNSUPPORTED = -3, -7, -1, -2, -5


@pytest.mark.parametrize("kw,code", [
    (dict(type=3), ARG), (dict(c_type=4), ARG), (dict(m=(1 << 24) + 1), UNSUPPORTED), (dict(lda=299), SHAPE), (dict(ldc=199), SHAPE),
    (dict(a_len=19 * 300 + 299), SHAPE), (dict(c_len=19 * 200 + 199), SHAPE), (dict(bias_len=199), SHAPE), (dict(act=3), ARG),
    (dict(a=0), NULL), (dict(c=0), NULL), (dict(a_by=2), ALIGN), (dict(c_by=2), ALIGN), (dict(space_len=-1), SHAPE), (dict(space=0), SHAPE),
    (dict(space_by=8), ALIGN), (dict(lda=1 << 61), SHAPE), (dict(c_is_a=True), ARG), (dict(space_is="a"), ARG), (dict(space_is="c"), ARG),
    (dict(m=0), 0), ({}, 0),
])
def test_products(tk, kw, code):
    import ctypes

    import numpy as np
    import torch

    import telmo_amd
    from telmo_amd import _lib
    from telmo_amd.kernels import _Epi

    m, k, n = 20, 300, 200
    w = telmo_amd.E4m3Weights.encode(tk, np.ones((n, k), np.float32), n, k)
    a, c = torch.ones(m * k + 4096, device="cuda"), torch.full((m * n + 4,), 5.0, device="cuda")
    need = w.workspace_bytes(m)
    space = torch.zeros(need + 64, dtype=torch.uint8, device="cuda")
    bias = torch.zeros(n, device="cuda")
    epi = _Epi(bias.data_ptr(), kw.get("bias_len", n), kw.get("act", 0), 1.0, 0)
    at = kw.get("a", a.data_ptr() + kw.get("a_by", 0))
    to = at if kw.get("c_is_a") else kw.get("c", c.data_ptr() + kw.get("c_by", 0))
    work = {"a": at, "c": to - to % 16}.get(kw.get("space_is"), kw.get("space", space.data_ptr() + kw.get("space_by", 0)))
    rc = _lib.lib().tg_linear_e4m3_device(tk._ctx, kw.get("type", 0), at, kw.get("a_len", m * k), kw.get("lda", k), kw.get("m", m),
                                          w._handle, kw.get("c_type", 0), to, kw.get("c_len", m * n), kw.get("ldc", n),
                                          ctypes.byref(epi), work, need + kw.get("space_len", 0))
    tk.synchronize()
    assert rc == code
    assert bool((c == 5.0).all()) or (code == 0 and kw.get("m", m))


def test_python_arguments(tk):
    import numpy as np
    import torch

    import telmo_amd

    w = telmo_amd.E4m3Weights.encode(tk, np.ones((32, 64), np.float32), 32, 64)
    a, c = torch.ones((4, 64), device="cuda"), torch.zeros((4, 32), device="cuda")
    for bad in (dict(a=a.double()), dict(a=a.cpu()), dict(c=c.int())):
        with pytest.raises(TypeError):
            tk.linear_e4m3_device(bad.get("a", a), w, bad.get("c", c))
    for bad in (dict(a=a[:, :63]), dict(c=c[:3]), dict(a=torch.ones((64, 4), device="cuda").t()), dict(c=c.t())):
        with pytest.raises(ValueError):
            tk.linear_e4m3_device(bad.get("a", a), w, bad.get("c", c))
    with pytest.raises(telmo_amd.TelmoError):
        tk.linear_e4m3_device(torch.ones((17, 64), device="cuda"), w, torch.zeros((17, 32), device="cuda"))
    values, scales = torch.zeros((200, 300), dtype=torch.uint8, device="cuda"), torch.ones((2, 3), device="cuda")
    for v, s in ((values.float(), scales), (values, scales.double()), (values, scales.cpu())):
        with pytest.raises(TypeError):
            telmo_amd.E4m3Weights.from_device(tk, v, s)
    for v, s in ((values, scales[:1]), (values.t(), scales)):
        with pytest.raises(ValueError):
            telmo_amd.E4m3Weights.from_device(tk, v, s)
    k = torch.zeros((7, 16, 2, 64), dtype=torch.uint8, device="cuda")
    e = torch.zeros((7, 2, 2), dtype=torch.int8, device="cuda")
    cache = telmo_amd.PagedCache(tk, k, k.clone(), k_exps=e, v_exps=e.clone())
    for x, y in ((e, None), (e, e[:6]), (e[:, :, :1], e[:, :, :1]), (torch.zeros((7, 3, 2), dtype=torch.int8, device="cuda"),) * 2):
        with pytest.raises(ValueError):
            telmo_amd.PagedCache(tk, k, k.clone(), k_exps=x, v_exps=y)
    for args in ((k.half(), k.half(), e, e), (k, k.clone(), e.int(), e.int())):
        with pytest.raises(TypeError):
            telmo_amd.PagedCache(tk, args[0], args[1], k_exps=args[2], v_exps=args[3])
    with pytest.raises(TypeError):
        telmo_amd.PagedCache(tk, k, k.clone())  # without exponents: no type of rows
    q = torch.zeros((1, 4, 32), device="cuda")
    with pytest.raises(ValueError):  # another head size
        telmo_amd.Attention(tk, 4, 32, kv_heads=2).paged(q, cache, torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                                                         torch.zeros(1, dtype=torch.int32, device="cuda"), q.clone())
