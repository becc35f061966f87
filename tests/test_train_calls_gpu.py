"""Ways to call the training operators that their documentation allows beside
the common ones: padded lengths given on the host in a captured call (refused),
the default stream's handle, very many and very large tensors."""
import numpy as np
import pytest

import raya_b200 as rb
from _train import close
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

def test_the_default_streams_handle(cuda_device):
    x, valid = make(2, 2, 150, 64, [150, 90], 62, 32)
    c = Call(x, valid, BLOCK3, 64, stream=0)
    c.forward()
    c.backward()
    got, want = c.results(), c.want()
    for n in want:
        close(got[n], want[n], n)


@pytest.mark.parametrize("batch,heads,seq,d", [(70000, 1, 3, 8), (3, 30000, 2, 136)])
def test_very_many_slices(cuda_device, batch, heads, seq, d):
    x, valid = make(batch, heads, seq, d, None, 63, 8)
    valid = np.random.default_rng(64).integers(0, seq + 1, batch)
    c = Call(x, valid, rb.Mask.FULL, 128, max_distance=3)
    c.forward()
    c.backward()
    got, want = c.results(), c.want()
    for n in want:
        close(got[n], want[n], n)


@pytest.mark.parametrize("heads,d,window", [(35, 64, 64), (18, 128, 64), (17, 136, 8)])
def test_offsets_beyond_32_bits(cuda_device, heads, d, window):
    """Tensors of more than 2^31 elements: the last head's results are those of a call on it alone."""
    import torch

    seq = 1 << 20
    assert heads * seq * d > 1 << 31
    params = rb.AttnParams(rb.Mask.sliding(window), 128, seq, 0.125)
    g = torch.Generator(device="cuda").manual_seed(65)
    x = torch.randn(1, heads, seq, d, generator=g, device="cuda")  # q, k, v and dout in one
    table = torch.randn(heads, 32, generator=g, device="cuda")
    valid = torch.tensor([seq - 777], dtype=torch.int32, device="cuda")

    def run(y, table):
        shape = rb.AttnShape(heads=y.shape[1], seq=seq, head_dim=d, batch=1)
        out, stats, bias = torch.empty_like(y), torch.empty(*y.shape[:3], 2, device="cuda"), rb.RelativeBias(table)
        rb.Cuda().attend_bias(shape, params, y, y, y, out, stats=stats, bias=bias, valid_len=valid)
        grads = [torch.empty_like(y) for _ in range(3)]
        dtable = torch.empty_like(table)
        rb.Cuda().attend_backward(shape, params, y, y, y, out, stats, y, *grads, bias=bias, dtable=dtable, valid_len=valid)
        return [z[:, -1:].clone() for z in (out, stats, *grads)] + [dtable[-1:].clone()]

    whole = run(x, table)
    one = run(x[:, -1:].contiguous(), table[-1:].contiguous())
    rb.sync_status()
    for n, a, b in zip(("out", "stats", "dq", "dk", "dv"), whole, one):
        assert torch.equal(a, b), n
        assert a[..., : seq - 777, :].abs().sum() > 0
    if d <= 128:  # above, the blocks of a slice, and with them the order of this sum, depend on the number of slices
        assert torch.equal(whole[-1], one[-1])
    del x, whole, one
    torch.cuda.empty_cache()
