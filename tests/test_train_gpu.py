"""The training operators on a B200 against their plain form in 64 bits
(tests/_train.py, which also derives the bounds): masks, odd lengths, padding
that holds NaN, rows without keys, biases that mask, magnitudes, streams,
captured graphs, and forward and backward run together as a step does."""
import math

import numpy as np
import pytest

import raya_b200 as rb
from _train import close, reference

pytestmark = pytest.mark.gpu

BLOCK3, OWN = rb.Mask.block(1), rb.Mask.block(0)


def make(batch, heads, seq, d, valid, seed, buckets=0, amp=1.0):
    rng = np.random.default_rng(seed)
    valid = np.full(batch, seq) if valid is None else np.asarray(valid)
    x = {n: rng.standard_normal((batch, heads, seq, d)).astype(np.float32) * np.float32(amp) for n in ("q", "k", "v", "dout")}
    x["dout"] *= np.float32(0.01)
    x["table"] = rng.standard_normal((heads, buckets)).astype(np.float32) if buckets else None
    return x, valid


class Call:
    """Forward and backward through the public calls; the padded rows of every input hold NaN, the outputs 7."""

    def __init__(self, x, valid, mask, block, max_distance=128, scale=None, stream=None):
        import torch

        b, h, s, d = x["q"].shape
        self.torch, self.x, self.valid_host, self.mask, self.block = torch, x, valid, mask, block
        self.max_distance, self.stream = max_distance, stream
        self.shape = rb.AttnShape(heads=h, seq=s, head_dim=d, batch=b)
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.scale = float(np.float32(self.scale))
        self.params = rb.AttnParams(mask, block, valid.tolist(), self.scale)
        pad = np.arange(s)[None, None, :, None] >= valid[:, None, None, None]
        self.t = {n: torch.from_numpy(np.where(pad, np.float32(np.nan), x[n])).cuda() for n in ("q", "k", "v", "dout")}
        self.bias = None
        if x["table"] is not None:
            self.bias = rb.RelativeBias(torch.from_numpy(x["table"]).cuda(), max_distance)
        self.valid = torch.from_numpy(valid.astype(np.int32)).cuda()
        full = lambda *n: torch.full(n, 7.0, device="cuda")  # noqa: E731
        self.t.update(out=full(b, h, s, d), stats=full(b, h, s, 2), dq=full(b, h, s, d), dk=full(b, h, s, d), dv=full(b, h, s, d))
        self.dtable = None if self.bias is None else torch.full_like(self.bias.table, 7.0)

    def forward(self, workspace=None):
        t = self.t
        rb.Cuda().attend_bias(self.shape, self.params, t["q"], t["k"], t["v"], t["out"], stats=t["stats"], bias=self.bias,
                              valid_len=self.valid, workspace=workspace, stream=self.stream)

    def poison(self):
        """NaN into the padded rows of what the backward pass reads."""
        pad = self.torch.arange(self.shape.seq, device="cuda")[None, None, :, None] >= self.valid[:, None, None, None]
        for n in ("out", "stats"):
            self.t[n] = self.t[n].masked_fill(pad, float("nan"))

    def backward(self, workspace=None):
        t = self.t
        rb.Cuda().attend_backward(self.shape, self.params, t["q"], t["k"], t["v"], t["out"], t["stats"], t["dout"], t["dq"],
                                  t["dk"], t["dv"], bias=self.bias, dtable=self.dtable, valid_len=self.valid,
                                  workspace=workspace, stream=self.stream)

    def results(self):
        rb.sync_status(self.stream)
        got = {n: self.t[n].cpu().numpy() for n in ("out", "dq", "dk", "dv")}
        st = self.t["stats"].cpu().numpy()
        got.update(m=st[..., :1], l=st[..., 1:])
        if self.dtable is not None:
            got["dtable"] = self.dtable.cpu().numpy()
        return got

    def want(self):
        x = self.x
        return reference(self.mask, self.block, self.scale, self.valid_host, x["q"], x["k"], x["v"], x["dout"], x["table"],
                         self.max_distance)


def check(x, valid, mask, block, **more):
    c = Call(x, valid, mask, block, **more)
    c.forward()
    first = c.results()
    c.poison()
    c.backward()
    got = {**c.results(), **{n: first[n] for n in ("out", "m", "l")}}  # as they were before poison()
    want = c.want()
    for n in ("out", "m", "l"):
        close(got[n], want[n], n)
    for n in ("dq", "dk", "dv") + (("dtable",) if x["table"] is not None else ()):
        close(got[n], want[n], n)
    pad = np.arange(c.shape.seq)[None, None, :] >= valid[:, None, None]
    pad = np.broadcast_to(pad, (c.shape.batch, c.shape.heads, c.shape.seq))
    for n, y in (("out", got["out"]), ("dq", got["dq"]), ("dk", got["dk"]), ("dv", got["dv"])):
        assert (y[pad] == 0).all() and not np.signbit(y[pad]).any(), f"{n}: padded rows are not +0"
    return c, got, want


CASES = [
    # batch, heads, seq, head_dim, valid, mask, block, buckets, max_distance
    (1, 1, 1, 64, None, BLOCK3, 128, 32, 128),
    (2, 1, 2, 64, [2, 1], rb.Mask.FULL, 128, 0, 0),
    (1, 2, 63, 64, None, rb.Mask.FULL, 128, 32, 128),
    (2, 2, 64, 64, [64, 33], rb.Mask.FULL, 128, 8, 16),
    (1, 2, 65, 64, None, BLOCK3, 64, 32, 128),
    (1, 1, 127, 64, None, rb.Mask.FULL, 128, 4, 2),
    (1, 2, 128, 64, None, OWN, 128, 32, 128),
    (2, 2, 129, 64, [129, 128], BLOCK3, 128, 32, 128),
    (3, 2, 300, 64, [300, 187, 0], BLOCK3, 64, 32, 128),
    (2, 3, 300, 64, [300, 1], rb.Mask.sliding(64), 128, 32, 128),
    (2, 1, 257, 64, [257, 200], rb.Mask.sliding(0), 128, 0, 0),
    (1, 2, 400, 64, None, rb.Mask.sliding(17), 128, 64, 300),
    (2, 2, 577, 64, [577, 500], rb.Mask.FULL, 128, 32, 128),
    (1, 1, 600, 64, None, rb.Mask.block(2), 32, 64, 600),
    (2, 2, 333, 64, [333, 100], OWN, 48, 30, 100),
    (1, 2, 200, 64, None, rb.Mask.block(1), 7, 32, 128),
    (1, 1, 1300, 64, None, BLOCK3, 256, 0, 0),
    (2, 2, 130, 8, [130, 77], BLOCK3, 64, 32, 128),
    (1, 2, 200, 40, None, rb.Mask.FULL, 128, 32, 128),
    (2, 1, 150, 56, [150, 149], rb.Mask.sliding(40), 128, 0, 0),
    (2, 2, 260, 96, [260, 130], rb.Mask.FULL, 128, 32, 128),
    (1, 2, 390, 128, None, BLOCK3, 128, 64, 256),
    (2, 1, 129, 72, [100, 129], rb.Mask.sliding(30), 128, 32, 128),
    (1, 2, 140, 136, None, BLOCK3, 64, 32, 128),
    (2, 1, 100, 256, [100, 41], rb.Mask.FULL, 128, 64, 4096),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in (c[:4] + (c[5].name(), c[6], c[7]))))
def test_forward_and_backward(cuda_device, case):
    batch, heads, seq, d, valid, mask, block, buckets, far = case
    x, valid = make(batch, heads, seq, d, valid, seq + d, buckets)
    check(x, valid, mask, block, max_distance=far or 128)


@pytest.mark.parametrize("d", [64, 96, 136])
def test_nothing_valid(cuda_device, d):
    x, valid = make(2, 2, 70, d, [0, 0], 5, 32)
    c, got, _ = check(x, valid, BLOCK3, 64)
    assert (got["dtable"] == 0).all()


@pytest.mark.parametrize("d", [64, 96, 136])
@pytest.mark.parametrize("masked", [-np.inf, np.finfo(np.float32).min, -(2.0 ** 100)])
def test_a_bias_that_masks(cuda_device, d, masked):
    """Buckets masked by -inf and by the lowest value: no weight, no gradient."""
    x, valid = make(2, 2, 210, d, [210, 150], 6, 16)
    x["table"][:, [0, 3, 9, 15]] = masked
    x["table"][1, :] = masked  # a head whose rows are all empty
    c, got, want = check(x, valid, rb.Mask.sliding(40), 128, max_distance=30)
    assert (got["dtable"][:, [0, 3, 9, 15]] == 0).all()
    assert (got["dq"][:, 1] == 0).all() and (got["dk"][:, 1] == 0).all() and (got["l"][:, 1] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 200])
def test_large_and_small_biases(cuda_device, d):
    x, valid = make(1, 2, 300, d, None, 8, 32)
    x["table"] *= np.float32(30)
    x["table"][:, 2] = 200.0  # one distance takes nearly all the weight
    x["table"][:, 20] = -300.0
    check(x, valid, BLOCK3, 64)


@pytest.mark.parametrize("amp", [2.0 ** -18, 1e-3, 30.0, 2.0 ** 12])
def test_magnitudes(cuda_device, amp):
    """Operands of any common size, past fp16's range: scores of ordinary size by the scale."""
    x, valid = make(1, 2, 260, 64, None, 9, 32, amp=amp)
    check(x, valid, BLOCK3, 64, scale=0.125 / amp ** 2)


def test_magnitudes_that_change_by_tile(cuda_device):
    x, valid = make(1, 2, 320, 64, None, 10)
    for n in ("k", "v", "dout", "q"):
        x[n] *= (2.0 ** (7 * (np.arange(320) // 64 % 3) - 7))[None, None, :, None].astype(np.float32)
    check(x, valid, rb.Mask.FULL, 128, scale=2.0 ** -14)


def test_sharp_softmax(cuda_device):
    """Scores of hundreds: nearly one key per row."""
    x, valid = make(2, 2, 190, 64, [190, 97], 11, 32, amp=6.0)
    check(x, valid, rb.Mask.FULL, 128)


def test_one_bad_row_stays_alone(cuda_device):
    """An infinite key is seen by the rows that its mask lets see it, and by no other."""
    x, valid = make(1, 1, 512, 64, None, 12)
    c = Call(x, valid, OWN, 64)
    c.t["k"][0, 0, 130, 5] = float("inf")
    c.forward()
    out = c.results()["out"][0, 0]
    rows = np.arange(512) // 64 == 130 // 64
    assert np.isfinite(out[~rows]).all() and not np.isfinite(out[rows]).all()
    clean = Call(x, valid, OWN, 64)
    clean.forward()
    assert np.array_equal(out[~rows], clean.results()["out"][0, 0][~rows])


@pytest.mark.parametrize("d", [64, 96, 136])
def test_equal_calls_give_equal_bits(cuda_device, d):
    x, valid = make(3, 3, 500, d, [500, 333, 64], 13, 32)
    a, b = (Call(x, valid, BLOCK3, 128) for _ in range(2))
    for c in (a, b):
        c.forward()
        c.backward()
    ra, rb_ = a.results(), b.results()
    for n in ra:
        assert np.array_equal(ra[n], rb_[n]), n


def test_one_sequence_of_a_batch_is_that_sequence(cuda_device):
    """A sequence's results do not depend on its place in a batch."""
    x, valid = make(3, 2, 300, 64, [300, 211, 90], 14)
    whole = Call(x, valid, BLOCK3, 64)
    whole.forward()
    whole.backward()
    got = whole.results()
    one = Call({n: None if y is None else y[1:2].copy() for n, y in x.items()}, valid[1:2], BLOCK3, 64)
    one.forward()
    one.backward()
    alone = one.results()
    for n in alone:
        assert np.array_equal(alone[n][0], got[n][1]), n


def test_no_bias_is_the_attention_of_attend_device(cuda_device):
    import torch

    x, valid = make(2, 3, 400, 64, [400, 222], 15)
    c = Call(x, valid, BLOCK3, 128)
    c.forward()
    out = torch.full_like(c.t["out"], 7.0)
    rb.Cuda().attend_device(c.shape, c.params, c.t["q"], c.t["k"], c.t["v"], out, valid_len=c.valid)
    want = c.want()["out"]
    close(out.cpu().numpy(), want, "attend_device")
    close(c.results()["out"], want, "attend_bias")


def test_optional_arguments(cuda_device):
    """No statistics, no gradient of the bias, lengths from params, a workspace of the caller's: the same values."""
    import torch

    x, valid = make(2, 2, 200, 64, [200, 77], 16, 32)
    c = Call(x, valid, BLOCK3, 64)
    c.forward()
    c.backward()
    got = c.results()
    t, k = c.t, rb.Cuda()
    out = torch.empty_like(t["out"])
    k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"], out, bias=c.bias)
    assert np.array_equal(out.cpu().numpy(), got["out"])
    size = rb.train_workspace(c.shape, c.params, c.bias, backward=True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    dq, dk, dv = (torch.empty_like(out) for _ in range(3))
    k.attend_backward(c.shape, c.params, t["q"], t["k"], t["v"], t["out"], t["stats"], t["dout"], dq, dk, dv, bias=c.bias,
                      workspace=ws)
    for n, y in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert np.array_equal(y.cpu().numpy(), got[n]), n
    with pytest.raises(rb.LengthError, match="workspace"):
        k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"], out, bias=c.bias, workspace=ws[:64])
    with pytest.raises(rb.LengthError, match="`dtable`"):
        k.attend_backward(c.shape, c.params, t["q"], t["k"], t["v"], t["out"], t["stats"], t["dout"], dq, dk, dv, bias=c.bias,
                          dtable=ws[:64].view(torch.float32))
    with pytest.raises(rb.LengthError, match="`stats`"):
        k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"], out, stats=t["stats"][:1])
    with pytest.raises(TypeError, match="`v`"):
        k.attend_bias(c.shape, c.params, t["q"], t["k"], t["v"].half(), out)
    with pytest.raises(TypeError, match="`k`"):
        k.attend_bias(c.shape, c.params, t["q"], t["k"].transpose(1, 2), t["v"], out)
    with pytest.raises(TypeError, match="dtable without a bias"):
        k.attend_backward(c.shape, c.params, t["q"], t["k"], t["v"], t["out"], t["stats"], t["dout"], dq, dk, dv,
                          dtable=c.dtable)
    with pytest.raises(rb.ShapeError, match="valid_len"):
        k.attend_bias(c.shape, rb.AttnParams(c.mask, 64, [200, 201], c.scale), t["q"], t["k"], t["v"], out)
    rb.sync_status()


@pytest.mark.parametrize("d", [64, 136])
def test_on_another_stream(cuda_device, d):
    """Work queued on a stream of the caller's, its inputs written there just before."""
    import torch

    x, valid = make(2, 2, 400, d, [400, 301], 17, 32)
    plain = Call(x, valid, BLOCK3, 64)
    plain.forward()
    plain.backward()
    want = plain.results()
    s = torch.cuda.Stream()
    c = Call(x, valid, BLOCK3, 64, stream=s)
    q = c.t["q"].clone()
    c.t["q"].zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        big = torch.ones(1 << 26, device="cuda")
        for _ in range(20):
            big.mul_(1.0)
        c.t["q"].copy_(q)
    c.forward()
    c.backward()
    got = c.results()
    for n in want:
        assert np.array_equal(got[n], want[n]), n


@pytest.mark.parametrize("d", [64, 136])
def test_captured_and_replayed(cuda_device, d):
    """Two captured steps of different lengths that share one workspace, replayed with new inputs."""
    import torch

    calls, graphs = [], []
    inputs = [make(2, 2, 300, d, [300, 150], 18, 32), make(1, 2, 200, d, None, 19, 32)]
    for x, valid in inputs:
        calls.append(Call(x, valid, BLOCK3, 64))
    size = max(rb.train_workspace(c.shape, c.params, c.bias, backward=True) for c in calls)
    size = max(size, *(rb.train_workspace(c.shape, c.params, c.bias) for c in calls))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    want = []
    for c in calls:
        c.forward(ws)
        c.backward(ws)
        want.append(c.results())
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.forward(ws)
            c.backward(ws)
        graphs.append(g)
    for c in calls:
        for n in ("out", "stats", "dq", "dk", "dv"):
            c.t[n].fill_(7.0)
        c.dtable.fill_(7.0)
    for turn in (0, 1, 0, 1):
        graphs[turn].replay()
    for c, w in zip(calls, want):
        got = c.results()
        for n in w:
            assert np.array_equal(got[n], w[n]), n
    calls[0].t["v"].mul_(2.0)
    graphs[0].replay()
    got = calls[0].results()
    assert np.array_equal(got["out"], 2 * want[0]["out"]) and np.array_equal(got["l"], want[0]["l"])


def test_captured_without_a_workspace_of_the_callers(cuda_device):
    import torch

    x, valid = make(2, 2, 200, 64, [200, 120], 20, 32)
    c = Call(x, valid, BLOCK3, 64)
    c.forward()
    c.backward()
    want = c.results()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.forward()
        c.backward()
    for n in ("out", "stats", "dq", "dk", "dv"):
        c.t[n].fill_(7.0)
    g.replay()
    got = c.results()
    for n in want:
        assert np.array_equal(got[n], want[n]), n


def test_a_training_step(cuda_device):
    """Forward, loss, backward and update of q, k, v and the table as a program runs them: along the gradient the loss
    changes as the gradients say."""
    import torch

    x, valid = make(2, 2, 260, 64, [260, 199], 21, 32)
    c = Call(x, valid, BLOCK3, 64)
    target = torch.from_numpy(np.random.default_rng(22).standard_normal(x["q"].shape).astype(np.float32)).cuda()
    rows = (torch.arange(260, device="cuda")[None, None, :, None] < c.valid[:, None, None, None])

    def loss():
        c.forward()
        return float((rows * (c.t["out"].double() - target) ** 2).sum() / 2)

    loss()
    c.t["dout"] = (rows * (c.t["out"] - target)).contiguous()
    c.backward()
    rb.sync_status()
    step = 1e-3
    leaves = [(c.t["q"], c.t["dq"]), (c.t["k"], c.t["dk"]), (c.t["v"], c.t["dv"]), (c.bias.table, c.dtable)]
    square = sum(float(g.double().square().sum()) for _, g in leaves)
    leaves = [(y, g.clone()) for y, g in leaves]
    at = []
    for sign in (1, -2):  # to + step, then to - step
        for y, g in leaves:
            y.add_(g, alpha=sign * step)
        at.append(loss())
    # L(+s) - L(-s) = 2 s g.g plus odd terms from s^3 on: the even ones cancel.  The table's gradient sums thousands of
    # pairs, so the quadratic term alone is ~0.08 of s g.g here, and the cubic one is of the order of its square.
    assert abs((at[0] - at[1]) / (2 * step) - square) < 0.05 * square, (at, square)


@pytest.mark.parametrize("heads,seq,d,far", [(2, 1500, 64, 4096), (1, 2000, 96, 4096), (1, 700, 64, 600)])
def test_distances_that_shared_memory_does_not_hold(cuda_device, heads, seq, d, far):
    """Bias tables whose distances are too many for a block's shared memory."""
    x, valid = make(1, heads, seq, d, [seq - 77], 23, 64)
    check(x, valid, rb.Mask.FULL, 128, max_distance=far)


def test_more_slices_than_one_chunk_of_the_workspace(cuda_device):
    """Images of more than the workspace holds at a time: every sequence as when called alone."""
    import torch

    batch, heads, seq = 20, 16, 8192  # 8 MB of images per slice, 2 GiB at a time
    shape = rb.AttnShape(heads=heads, seq=seq, head_dim=64, batch=batch)
    params = rb.AttnParams(BLOCK3, 128, seq, 0.125)
    g = torch.Generator(device="cuda").manual_seed(24)
    t = {n: torch.randn(batch, heads, seq, 64, generator=g, device="cuda") for n in ("q", "k", "v", "dout")}
    bias = rb.RelativeBias(torch.randn(heads, 32, generator=g, device="cuda"))
    valid = torch.randint(1000, seq + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)

    def run(at):
        x = {n: y[at] for n, y in t.items()}
        sh = rb.AttnShape(heads=heads, seq=seq, head_dim=64, batch=x["q"].shape[0])
        out, stats = torch.empty_like(x["q"]), torch.empty(*x["q"].shape[:3], 2, device="cuda")
        rb.Cuda().attend_bias(sh, params, x["q"], x["k"], x["v"], out, stats=stats, bias=bias, valid_len=valid[at])
        grads = [torch.empty_like(out) for _ in range(3)]
        dtable = torch.empty_like(bias.table)
        rb.Cuda().attend_backward(sh, params, x["q"], x["k"], x["v"], out, stats, x["dout"], *grads, bias=bias, dtable=dtable,
                                  valid_len=valid[at])
        return [out, stats, *grads, dtable]

    need = rb.train_workspace(shape, params, bias, backward=True)
    assert need < 3 << 30 and need < batch * heads * 8 << 20  # one chunk at a time
    whole = run(slice(0, batch))
    table = torch.zeros_like(bias.table, dtype=torch.float64)
    for b in range(batch):
        one = run(slice(b, b + 1))
        for x, y in zip(whole[:-1], one[:-1]):
            assert torch.equal(x[b : b + 1], y), b
        table += one[-1].double()
    # each sequence's gradient is rounded to fp32 once, and the whole's
    assert ((whole[-1] - table).abs() <= 2.0 ** -24 * (batch + 1) * table.abs().max()).all()
    rb.sync_status()


@pytest.mark.parametrize("d", [64, 96, 136])
def test_two_calls_at_once(cuda_device, d):
    """Calls on two streams, each with a workspace of its own, in each other's way on the SMs."""
    import torch

    inputs = [make(2, 4, 700, d, [700, 401], 25, 32), make(3, 2, 500, d, [500, 33, 444], 26)]
    want = []
    for x, valid in inputs:
        c = Call(x, valid, BLOCK3, 64)
        c.forward()
        c.backward()
        want.append(c.results())
    streams = [torch.cuda.Stream() for _ in inputs]
    calls = [Call(x, valid, BLOCK3, 64, stream=s) for (x, valid), s in zip(inputs, streams)]
    torch.cuda.synchronize()
    for _ in range(20):
        for c in calls:
            c.forward()
            c.backward()
    for c, w in zip(calls, want):
        got = c.results()
        for n in w:
            assert np.array_equal(got[n], w[n]), n


@pytest.mark.parametrize("d", [64, 96, 136])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales_that_turn_or_drop_the_scores(cuda_device, d, scale):
    x, valid = make(2, 2, 150, d, [150, 65], 27, 32)
    check(x, valid, BLOCK3, 64, scale=scale)


@pytest.mark.parametrize("d", [64, 96, 136])
def test_lengths_outside_the_sequence_are_clamped(cuda_device, d):
    import torch

    x, valid = make(3, 2, 140, d, [140, 0, 77], 28, 32)
    calls = [Call(x, valid, BLOCK3, 64) for _ in range(2)]
    calls[1].valid = torch.tensor([2 ** 31 - 1, -5, 77], dtype=torch.int32, device="cuda")
    for c in calls:
        c.forward()
        c.backward()
    want, got = (c.results() for c in calls)
    for n in want:
        assert np.array_equal(got[n], want[n]), n


@pytest.mark.parametrize("d", [64, 136])
@pytest.mark.parametrize("mask,block", [(rb.Mask.block(2 ** 31 - 1), 64), (rb.Mask.block(0), 2 ** 31 - 1),
                                        (rb.Mask.sliding(2 ** 31 - 1), 128), (rb.Mask.block(1), 1)])
def test_masks_at_their_limits(cuda_device, mask, block, d):
    x, valid = make(2, 2, 200, d, [200, 131], 29, 32)
    check(x, valid, mask, block)


@pytest.mark.parametrize("batch,heads,seq", [(300, 1, 70), (1, 200, 3), (40, 5, 1)])
def test_many_short_slices(cuda_device, batch, heads, seq):
    x, valid = make(batch, heads, seq, 64, None, 30, 32)
    valid = np.random.default_rng(31).integers(0, seq + 1, batch)
    check(x, valid, BLOCK3, 64)


@pytest.mark.parametrize("d", [64, 96, 136])
def test_one_tensor_in_several_places(cuda_device, d):
    """q, k and v (and dout and out) may be the same tensor: nothing reads what another has written."""
    x, valid = make(1, 2, 190, d, None, 32, 32)
    x["k"] = x["v"] = x["q"]
    c = Call(x, valid, BLOCK3, 64)
    c.t["k"] = c.t["v"] = c.t["q"]
    c.forward()
    c.x["dout"] = c.t["out"].cpu().numpy()
    c.t["dout"] = c.t["out"]
    c.backward()
    got, want = c.results(), c.want()
    for n in want:
        close(got[n], want[n], n)


def test_a_stream_handle_and_a_workspace_of_floats(cuda_device):
    """The stream as the integer that other libraries hand out, views that start past their storage, a larger workspace
    of another type, and a bias whose gradient nobody asks for."""
    import torch

    x, valid = make(2, 2, 200, 64, [200, 77], 33, 32)
    c = Call(x, valid, BLOCK3, 64)
    c.forward()
    c.backward()
    want = c.results()
    s = torch.cuda.Stream()
    size = rb.train_workspace(c.shape, c.params, c.bias, backward=True)
    ws = torch.empty(size // 4 + 1000, device="cuda")
    d = Call(x, valid, BLOCK3, 64, stream=s.cuda_stream)
    for n, y in d.t.items():
        room = torch.empty(y.numel() + 4, device="cuda")
        room[4:].copy_(y.reshape(-1))
        d.t[n] = room[4:].view(y.shape)
    torch.cuda.synchronize()
    d.forward(ws)
    d.dtable = None
    d.backward(ws)
    got = d.results()
    for n in got:
        assert np.array_equal(got[n], want[n]), n
