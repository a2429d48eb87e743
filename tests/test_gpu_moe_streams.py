"""MoeLayer calls with stream=: what they return is not memory that the current stream still writes to."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_results_on_another_stream_have_memory_of_their_own(native):
    from loki_b200.moe import LayerWeights, MoeLayer
    W, layer = LayerWeights("cuda", 1, 0), MoeLayer(0, max_tokens=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, resid = torch.randn(4, 7168, generator=g, device="cuda"), torch.randn(4, 7168, generator=g, device="cuda")
    _, sel, w = layer.route(W, x)

    def calls(stream):
        yield lambda: layer.forward(W, x, resid, stream=stream)
        yield lambda: layer.route(W, x, stream=stream)
        yield lambda: layer.dispatch(sel, w, stream=stream)
        yield lambda: layer.experts(W, x, resid, sel, w, stream=stream)
    s = torch.cuda.Stream()
    for plain, other in zip(calls(None), calls(s)):
        want = [t.clone() for t in plain()]
        torch.cuda.synchronize()
        other()                                                          # the stream's pool has seen such a call
        torch.cuda.synchronize()
        for t in want:                                                   # given back with a write still in the current stream's queue
            held = torch.empty_like(t)
            torch.cuda._sleep(200_000_000)
            held.fill_(7)
            del held
        got = other()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    layer.device_error()
    layer.close()
