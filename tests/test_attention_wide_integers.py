"""Positions past 64 bits, without a GPU: ctypes would cut them to other positions."""
import pytest


class Kern:
    device = -1  # get_device of a host tensor


@pytest.mark.parametrize("far", (2**62, 2**63, 2**64, 2**64 + 5, 10**30))
def test_windows_past_64_bits_have_no_limit(far):
    from telmo_amd import attention

    desc = attention.Attention(Kern, 2, 64, left=far, right=far)._desc
    assert desc.left >= 2**62 and desc.right >= 2**62


@pytest.mark.parametrize("start", (2**63, 2**64, -2**64))
def test_starts_past_64_bits_are_refused(start):
    import torch

    from telmo_amd import attention

    rotary, x = attention.Rotary.__new__(attention.Rotary), torch.zeros(3, 2, 64)
    rotary._kernels = Kern
    with pytest.raises(ValueError, match="start"):
        rotary.apply(x, x, start=start)
