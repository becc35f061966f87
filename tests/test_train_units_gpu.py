"""The training operators where every CTA takes several units of work: the
persistent kernels run two CTAs on an SM for head_dim up to 64 and one for 72
to 128, so these calls have at least twice as many 128-row units as CTAs.
Compared with the plain form in 64 bits (tests/_train.py), and with
themselves: a row of one unit that got a value of another would show in both."""
import numpy as np
import pytest

import raya_b200 as rb
from _train import close
from test_train_gpu import Call, make

pytestmark = pytest.mark.gpu

OWN, WINDOW, FULL = rb.Mask.block(0), rb.Mask.sliding(40), rb.Mask.FULL
SMS = 148


def lengths(batch, seq, seed):
    """Uneven, most of them past the last unit's first row; the first ones whole, empty and of one row."""
    rng = np.random.default_rng(seed)
    valid = rng.integers((seq - 1) // 128 * 128 + 1, seq + 1, batch)
    valid[:3] = seq, 0, 1
    return valid


def units(valid, heads):
    return int(((valid + 127) // 128).sum()) * heads


CASES = [
    # batch, heads, seq, head_dim, mask, block, buckets, whether the table's gradient is asked for
    (80, 8, 64, 64, OWN, 64, 0, False),  # one 64-column tile a unit
    (80, 8, 64, 64, OWN, 64, 32, True),
    (80, 8, 200, 64, OWN, 64, 32, False),
    (80, 8, 150, 64, WINDOW, 128, 0, False),
    (80, 8, 150, 64, WINDOW, 128, 32, True),
    (80, 8, 150, 64, FULL, 128, 0, False),
    (80, 8, 150, 64, FULL, 128, 32, False),
    (80, 8, 150, 64, FULL, 128, 32, True),
    (40, 8, 300, 64, rb.Mask.block(1), 64, 32, True),
    (80, 8, 140, 40, WINDOW, 128, 16, True),
    (80, 8, 70, 8, FULL, 128, 0, False),
    (40, 8, 64, 96, OWN, 64, 0, False),
    (40, 8, 64, 96, OWN, 64, 32, True),
    (40, 8, 150, 96, WINDOW, 128, 32, False),
    (40, 8, 150, 96, FULL, 128, 0, False),
    (40, 8, 150, 72, FULL, 128, 64, True),
    (40, 8, 64, 128, OWN, 64, 0, False),
    (40, 8, 64, 128, OWN, 64, 32, True),
    (40, 8, 150, 128, WINDOW, 128, 0, False),
    (40, 8, 150, 128, WINDOW, 128, 32, True),
    (40, 8, 150, 128, FULL, 128, 32, False),
    (20, 8, 300, 128, rb.Mask.block(1), 64, 32, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:4] + (c[4].name(),) + c[5:]))
def test_several_units_per_cta(cuda_device, case):
    import torch

    batch, heads, seq, d, mask, block, buckets, grad = case
    assert torch.cuda.get_device_properties(0).multi_processor_count == SMS
    valid = lengths(batch, seq, seq + d)
    assert units(valid, heads) >= 2 * SMS * (2 if d <= 64 else 1)
    x, valid = make(batch, heads, seq, d, valid, seq + d + 1, buckets)
    c = Call(x, valid, mask, block)
    if not grad:
        c.dtable = None
    c.forward()
    first = c.results()
    c.poison()
    c.backward()
    got = {**c.results(), **{n: first[n] for n in ("out", "m", "l")}}
    want = c.want()
    for n in ("out", "m", "l", "dq", "dk", "dv") + (("dtable",) if grad else ()):
        close(got[n], want[n], n)
    pad = np.broadcast_to(np.arange(seq)[None, None, :] >= valid[:, None, None], (batch, heads, seq))
    for n in ("out", "dq", "dk", "dv"):
        assert (got[n][pad] == 0).all() and not np.signbit(got[n][pad]).any(), f"{n}: padded rows are not +0"
    for _ in range(3):
        for n in ("out", "dq", "dk", "dv"):
            c.t[n].fill_(7.0)
        c.forward()
        c.backward()
        again = c.results()
        for n in ("out", "dq", "dk", "dv") + (("dtable",) if grad else ()):
            assert np.array_equal(again[n], got[n]), n


@pytest.mark.parametrize("batch,heads,seq,d", [(1, 12, 512, 64), (40, 8, 150, 64), (2, 8, 300, 96), (1, 2, 90, 136)])
def test_the_tables_gradient_in_a_workspace_with_old_contents(cuda_device, batch, heads, seq, d):
    """Calls on different inputs one behind the other in one workspace, which first holds NaN: the last sum, which is
    launched before the partials are complete, finds those of its own call."""
    import torch

    calls, want = [], []
    for seed in (41, 42):
        x, valid = make(batch, heads, seq, d, None, seed, 32)
        c = Call(x, valid, rb.Mask.block(1), 64)
        c.forward()
        c.backward()
        want.append(c.results())
        close(want[-1]["dtable"], c.want()["dtable"], "dtable")
        calls.append(c)
    ws = torch.full((rb.train_workspace(c.shape, c.params, c.bias, backward=True),), 255, dtype=torch.uint8, device="cuda")
    sums = []
    for turn in range(20):
        c = calls[turn % 2]
        c.dtable.fill_(7.0)
        c.backward(ws)
        sums.append(c.dtable.clone())
    rb.sync_status()
    for turn, y in enumerate(sums):
        assert np.array_equal(y.cpu().numpy(), want[turn % 2]["dtable"]), turn


@pytest.mark.parametrize("batch,heads,seq,d,buckets", [(1, 2, 512, 64, 0), (1, 12, 512, 64, 32), (80, 8, 150, 64, 0),
                                                       (2, 8, 300, 96, 0), (40, 8, 150, 128, 32)])
def test_gradients_in_a_workspace_of_ones(cuda_device, batch, heads, seq, d, buckets):
    """The workspace holds 1 in every word, then what calls on other inputs left: the gradients of k and v, whose kernels
    start before the one ahead of them is complete, are those of their own call."""
    import torch

    calls, want = [], []
    for seed in (43, 44):
        x, valid = make(batch, heads, seq, d, None, seed, buckets)
        c = Call(x, valid, rb.Mask.block(1), 64)
        c.forward()
        c.backward()
        got, full = c.results(), c.want()
        for n in ("dq", "dk", "dv"):
            close(got[n], full[n], n)
        want.append(got)
        calls.append(c)
    ws = torch.ones(rb.train_workspace(c.shape, c.params, c.bias, backward=True) // 4, dtype=torch.int32, device="cuda")
    for fresh in (True, False):
        for turn in range(12):
            c = calls[turn % 2]
            for n in ("dq", "dk", "dv"):
                c.t[n].fill_(7.0)
            if fresh:
                ws.fill_(1)
            c.backward(ws)
            got = c.results() if fresh or turn >= 10 else None
            for n in ("dq", "dk", "dv") if got else ():
                assert np.array_equal(got[n], want[turn % 2][n]), (n, turn)
