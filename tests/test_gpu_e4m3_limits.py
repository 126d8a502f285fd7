"""The largest calls of the product in eight bits: what is refused leaves nothing behind."""
import pytest

pytestmark = pytest.mark.gpu

UNSUPPORTED = -5


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
    assert rc == UNSUPPORTED
    assert bool((space == 0xA5).all())
    # An allocator's leftovers are not for the tests after this one.
    del a, space
    torch.cuda.empty_cache()
