"""A Rotary's frequencies outlive it, on an MI355X."""
import gc
import weakref

import pytest

pytestmark = pytest.mark.gpu


def test_a_rotary_may_go_while_its_calls_are_queued(gpu_stream):
    """On another stream than torch's, behind work that holds it up: what torch hands out meanwhile does not lie
    where the queued kernels read their frequencies."""
    import torch

    import telmo_amd

    stream = torch.cuda.Stream()
    kern = telmo_amd.Kernels(0, stream=stream.cuda_stream)
    x = torch.randn(50, 3, 64, device="cuda")
    want, got, others = torch.zeros_like(x), [torch.zeros_like(x) for _ in range(4)], []
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    kept = telmo_amd.Rotary(kern, 64, base=500.0)
    kept.apply(x, want, start=9)
    kern.synchronize()
    kern2 = telmo_amd.Kernels(0, stream=stream.cuda_stream)
    for out in got:
        with torch.cuda.stream(stream):
            for _ in range(10):
                torch.mm(big, big)
        rotary = telmo_amd.Rotary(kern2, 64, base=500.0)
        rotary.apply(x, out, start=9)
        turns = weakref.ref(rotary.turns)
        del rotary
        gc.collect()
        assert turns() is not None
        others += [torch.full((32,), 0.25, dtype=torch.float64, device="cuda") for _ in range(50)]
    torch.cuda.synchronize()
    for out in got:
        assert torch.equal(out, want)
    for k in (kern, kern2):
        k.close()


def test_rotaries_of_one_context_share_their_frequencies(tk):
    import telmo_amd

    a, b, c = (telmo_amd.Rotary(tk, 64, base=base, interleaved=i) for base, i in ((100.0, False), (100.0, True), (101.0, False)))
    assert a.turns is b.turns and a.turns is not c.turns
