"""A decode on one thread while another one captures a graph, on an MI355X."""
import threading

import numpy as np
import pytest

from helpers import tdt_network
from test_gpu_tdt import DECODE_CASES, TOL, say, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams", (1, 3))
def test_a_decode_runs_while_another_thread_captures(orc, gpu_stream, streams):
    """The capture stays open until the decode has returned its tokens: both stand."""
    import torch

    import telmo_amd

    h, vocab, durs, layers, p, frames, blank_bias, ms = DECODE_CASES[4]
    rng = np.random.default_rng(310)
    net = tdt_network(rng, h, vocab, durs, layers=layers, precision=p, max_symbols=ms, blank_bias=blank_bias)
    enc = rng.standard_normal((frames, h)).astype(np.float32)
    state = (0.3 * rng.standard_normal(layers * 2 * h)).astype(np.float32)
    pred = (0.3 * rng.standard_normal(h)).astype(np.float32)
    want_state, want_pred = state.copy(), pred.copy()
    tokens, frame, on = orc.tdt_decode(net, enc, want_state, want_pred)
    kern = telmo_amd.Kernels(0)
    dec = upload(kern, net)
    encs = [torch.from_numpy(enc).cuda() for _ in range(streams)]
    rounds = [[(torch.from_numpy(state.copy()).cuda(), torch.from_numpy(pred.copy()).cuda()) for _ in range(streams)]
              for _ in range(2)]
    x, graph, stream = torch.ones(1000, device="cuda"), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    open_, done, results, errors = threading.Event(), threading.Event(), [], []

    def decode(buffers):
        if streams == 1:
            return [dec.decode(encs[0], *buffers[0])]
        return dec.decode_streams(encs, [s for s, _ in buffers], [q for _, q in buffers])

    def run():
        try:
            open_.wait(60)
            results.append(decode(rounds[1]))
        except Exception as e:  # reported by the main thread
            errors.append(e)
        finally:
            done.set()

    say("decode beside a capture", streams)
    decode(rounds[0])  # what the decoder allocates on its first call
    thread = threading.Thread(target=run)
    thread.start()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        x.mul_(2.0)
        open_.set()
        assert done.wait(60)
        x.add_(1.0)
    thread.join(60)
    assert not errors, errors
    kern.synchronize()
    for (toks, got_frame, got_on), (s, _) in zip(results[0], rounds[1]):
        assert [tuple(t) for t in toks] == tokens and (got_frame, got_on) == (frame, on)
        assert np.max(np.abs(s.cpu().numpy() - want_state)) <= TOL
    for value in (3.0, 7.0, 15.0):
        graph.replay()
        torch.cuda.synchronize()
        assert bool((x == value).all())
    dec.close()
    kern.close()
