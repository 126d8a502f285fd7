"""The largest calls of the product in eight bits: what is refused leaves nothing behind."""
import pytest

pytestmark = pytest.mark.gpu

UNSUPPORTED, NOMEM = -5, -6


def test_too_many_tiles_leave_the_workspace_alone(tk):
    """2^24 rows by 16384 outputs are 2^24 tiles. The outputs' address is never used."""
    import torch

    import telmo_amd
    from telmo_amd import _lib

    m, k, n = 1 << 24, 1, 16384
    w = telmo_amd.E4m3Weights.from_device(tk, torch.zeros((n, k), dtype=torch.uint8, device="cuda"), torch.ones((n // 128, 1), device="cuda"))
    a = torch.ones(m * k, device="cuda")
    space = torch.full((w.workspace_bytes(m),), 0xA5, dtype=torch.uint8, device="cuda")
    tk.synchronize()
    rc = _lib.lib().tg_linear_e4m3_device(tk._ctx, 0, a.data_ptr(), a.numel(), k, m, w._handle, 0, 1 << 50, m * n, n, None,
                                          space.data_ptr(), space.numel())
    tk.synchronize()
    left_alone = bool((space == 0xA5).all())  # not in the assertion, whose report would take the tensor apart
    del a, space
    torch.cuda.empty_cache()
    assert rc == UNSUPPORTED and left_alone


def test_many_rows_without_inputs(tk):
    """The epilogue of empty sums, for more rows than a launch's second dimension has workgroups."""
    import torch

    import telmo_amd

    m, n = (1 << 22) + 5, 3
    w = telmo_amd.E4m3Weights.from_device(tk, torch.zeros((n, 0), dtype=torch.uint8, device="cuda"), torch.zeros((1, 0), device="cuda"))
    a, c = torch.zeros((m, 0), device="cuda"), torch.full((m + 1, n), 2.0, device="cuda")
    bias = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    space = torch.zeros(w.workspace_bytes(m), dtype=torch.uint8, device="cuda")
    tk.linear_e4m3_device(a, w, c[:m], telmo_amd.Epilogue(bias=bias, scale=0.5), workspace=space)
    tk.synchronize()
    assert torch.equal(c[:m], (0.5 * bias).expand(m, n)) and bool((c[m] == 2.0).all())


def test_many_rows_of_few_inputs(tk):
    """More rows than the rounding has workgroups for at a time: whole numbers, which e4m3 and the sums hold exactly."""
    import torch

    import telmo_amd

    m, k, n = (1 << 22) + 5, 2, 3
    values = torch.tensor([[0x38, 0x40], [0x40, 0x38], [0x38, 0xB8]], dtype=torch.uint8, device="cuda")  # 1 2, 2 1, 1 -1
    w = telmo_amd.E4m3Weights.from_device(tk, values, torch.ones((1, 1), device="cuda"))
    a = (torch.arange(m * k, device="cuda") % 17 - 8).float().reshape(m, k)
    c = torch.full((m + 1, n), 2.0, device="cuda")
    space = torch.zeros(w.workspace_bytes(m), dtype=torch.uint8, device="cuda")
    tk.linear_e4m3_device(a, w, c[:m], workspace=space)
    tk.synchronize()
    x, y = a[:, 0], a[:, 1]
    assert torch.equal(c[:m], torch.stack([x + 2 * y, 2 * x + y, x - y], 1)) and bool((c[m] == 2.0).all())


def test_weights_that_do_not_fit_leave_no_error_behind(tk):
    """2^48 bytes of weights: the allocation fails before anything is read, and the next call is none the worse."""
    import ctypes

    import torch

    import telmo_amd
    from telmo_amd import _lib

    n = 1 << 24
    w = telmo_amd.E4m3Weights.from_device(tk, torch.zeros((16, 16), dtype=torch.uint8, device="cuda"), torch.ones((1, 1), device="cuda"))
    a, c = torch.ones((1, 16), device="cuda"), torch.full((1, 16), 2.0, device="cuda")
    small, out = (ctypes.c_uint8 * 16)(), ctypes.c_void_p()
    for upload, at in ((_lib.lib().tg_weights_e4m3_upload, ctypes.addressof(small)), (_lib.lib().tg_weights_e4m3_upload_device, a.data_ptr())):
        assert upload(tk._ctx, at, n * n, n, at, (n // 128)**2, n, n, ctypes.byref(out)) == NOMEM and not out.value
        tk.linear_e4m3_device(a, w, c)
        tk.synchronize()
        assert bool((c == 0).all())


def test_other_weights_that_do_not_fit_leave_no_error_behind(tk):
    """The same of int8 weights, 2^48 bytes of them too."""
    import ctypes

    import torch

    import telmo_amd
    from telmo_amd import _lib

    w = telmo_amd.E4m3Weights.from_device(tk, torch.zeros((16, 16), dtype=torch.uint8, device="cuda"), torch.ones((1, 1), device="cuda"))
    a, c = torch.ones((1, 16), device="cuda"), torch.full((1, 16), 2.0, device="cuda")
    small, out = (ctypes.c_uint8 * 16)(), ctypes.c_void_p()
    n = 1 << 24
    at = ctypes.addressof(small)
    rc = _lib.lib().tg_weights_upload(tk._ctx, at, n * n, at, n, int(telmo_amd.Precision.INT8), n, n, ctypes.byref(out))
    assert rc == NOMEM and not out.value
    tk.linear_e4m3_device(a, w, c)
    tk.synchronize()
    assert bool((c == 0).all())
