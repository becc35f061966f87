"""Ways to call the training operators that their documentation allows beside
the common ones: padded lengths given on the host in a captured call (refused)."""
import numpy as np
import pytest

import raya_b200 as rb
from test_train_gpu import BLOCK3, Call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("on_stream", [False, True])
def test_host_lengths_in_a_captured_call_are_refused(cuda_device, on_stream):
    """Uploading them would wait for the stream, which a capture cannot: refused before anything is queued, and the
    capture goes on."""
    import torch

    x, valid = make(2, 2, 150, 64, [150, 90], 61, 32)
    c = Call(x, valid, BLOCK3, 64)
    c.forward()
    want = c.results()["out"]
    t, k = c.t, rb.Cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stream = torch.cuda.current_stream().cuda_stream if on_stream else None
        with pytest.raises(rb.UnsupportedError, match="captured"):
            k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"], t["out"], stats=t["stats"], bias=c.bias, stream=stream)
        c.forward()
    t["out"].fill_(7.0)
    g.replay()
    assert np.array_equal(c.results()["out"], want)
    out = torch.full_like(t["out"], 7.0)
    k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"], out, stats=t["stats"], bias=c.bias)
    assert np.array_equal(out.cpu().numpy(), want)

