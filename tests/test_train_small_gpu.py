"""Gradients of keys that every query weighs little, and of rows far smaller
than their neighbours, within the bounds of tests/_train_tight.py: relative to
each result's own size, as fp32 arithmetic gives them."""
import numpy as np
import pytest

import raya_b200 as rb
from _train import close
from _train_tight import tight
from test_train_gpu import BLOCK3, CASES, Call, make

pytestmark = pytest.mark.gpu

GRADIENTS = ("dv", "dk", "dq")


def run(x, valid, mask, block, **more):
    c = Call(x, valid, mask, block, **more)
    c.forward()
    c.poison()
    c.backward()
    return c, c.results()


def want_of(c):
    x = c.x
    return tight(c.mask, c.block, c.scale, c.valid_host, x["q"], x["k"], x["v"], x["dout"], x["table"], c.max_distance)


def weak_keys(d, bits, seed, seq=190, buckets=0, amount=3):
    """Keys whose scores lie `bits` powers of two below the others in every row: the first column of q is 4, that of
    such a key what brings its score down."""
    x, valid = make(2, 2, seq, d, [seq, seq - 30], seed, buckets)
    x["q"][..., 0], x["k"][..., 0] = 4.0, 0.0
    weak = np.array([5, 40, 77, 100, 130, 150][:amount])
    x["k"][:, :, weak, 0] = -bits * np.log(2.0) * np.sqrt(d) / 4.0
    return x, valid, weak


@pytest.mark.parametrize("d", [64, 40, 96, 128, 136])
@pytest.mark.parametrize("bits", [20, 28, 36, 60, 100])
def test_the_value_gradient_of_keys_with_small_weights(cuda_device, d, bits):
    x, valid, weak = weak_keys(d, bits, 51, buckets=32 if bits == 36 else 0)
    c, got = run(x, valid, rb.Mask.FULL, 128)
    value, bound = want_of(c)["dv"]
    size = np.abs(value[:, :, weak]).max(-1, keepdims=True)
    assert (size > 0).all() and (bound[:, :, weak] < 4e-3 * size).all()  # the bound asks for something here
    close(got["dv"], (value, bound), "dv")


@pytest.mark.parametrize("mask,block", [(rb.Mask.sliding(40), 128), (BLOCK3, 64), (rb.Mask.block(0), 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_value_gradients_of_small_weights_under_masks(cuda_device, mask, block, d):
    """Weak and ordinary keys side by side in a tile, with blocks that the mask leaves empty."""
    x, valid, weak = weak_keys(d, 50, 52, seq=330, amount=6)
    c, got = run(x, valid, mask, block)
    close(got["dv"], want_of(c)["dv"], "dv")


@pytest.mark.parametrize("d", [64, 40, 96, 128, 136])
@pytest.mark.parametrize("bits", [20, 28, 36, 60, 100])
def test_the_key_gradient_of_keys_with_small_weights(cuda_device, d, bits):
    x, valid, weak = weak_keys(d, bits, 53, buckets=32 if bits == 36 else 0)
    c, got = run(x, valid, rb.Mask.FULL, 128)
    value, bound = want_of(c)["dk"]
    size = np.abs(value[:, :, weak]).max(-1, keepdims=True)
    assert (size > 0).all() and (bound[:, :, weak] < 0.25 * size).all()
    close(got["dk"], (value, bound), "dk")


@pytest.mark.parametrize("mask,block", [(rb.Mask.sliding(40), 128), (BLOCK3, 64), (rb.Mask.block(0), 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_key_gradients_of_small_weights_under_masks(cuda_device, mask, block, d):
    x, valid, weak = weak_keys(d, 50, 54, seq=330, amount=6)
    c, got = run(x, valid, mask, block)
    close(got["dk"], want_of(c)["dk"], "dk")


@pytest.mark.parametrize("d", [64, 128])
def test_weak_keys_of_units_behind_the_first(cuda_device, d):
    """The same where each CTA takes several units, some with weak keys and some without."""
    batch, seq = (80, 150) if d == 64 else (40, 150)
    x, valid = make(batch, 8, seq, d, None, 55)
    x["q"][..., 0], x["k"][..., 0] = 4.0, 0.0
    x["k"][1::3, :, [3, 70, 140], 0] = -45 * np.log(2.0) * np.sqrt(d) / 4.0
    c, got = run(x, valid, rb.Mask.FULL, 128)
    want = want_of(c)
    for n in GRADIENTS:
        close(got[n], want[n], n)


@pytest.mark.parametrize("d", [64, 96, 136])
def test_gradients_that_are_zero_but_for_a_few_rows(cuda_device, d):
    """dout of one row only, and of none: keys whose queries have no gradient, next to some that do."""
    x, valid = make(2, 2, 300, d, [300, 170], 56, 32)
    for rows in ([7], [], [69, 150]):
        dout = np.zeros_like(x["dout"])
        dout[:, :, rows] = x["dout"][:, :, rows]
        y = dict(x, dout=dout)
        c, got = run(y, valid, BLOCK3, 64)
        want = want_of(c)
        for n in GRADIENTS + ("dtable",):
            close(got[n], want[n], n)
            assert rows or (got[n] == 0).all()


@pytest.mark.parametrize("d", [64, 40, 128, 136])
@pytest.mark.parametrize("live", [[7, 69, 150], [70, 71], [3]])
def test_weak_keys_of_the_rows_that_have_a_gradient(cuda_device, d, live):
    """As in training on some tokens only: the other rows' dout is zero, and it is they that weigh the keys highly."""
    x, valid = make(2, 2, 200, d, [200, 155], 59)
    weak = [5, 77, 130]
    x["q"][..., 0], x["k"][..., 0] = 0.0, 0.0
    x["q"][:, :, live, 0] = 4.0
    x["k"][:, :, weak, 0] = -45 * np.log(2.0) * np.sqrt(d) / 4.0
    dout = np.zeros_like(x["dout"])
    dout[:, :, live] = x["dout"][:, :, live]
    x["dout"] = dout
    c, got = run(x, valid, rb.Mask.FULL, 128)
    want = want_of(c)
    size = np.abs(want["dv"][0][:, :, weak]).max(-1, keepdims=True)
    assert (size[0] > 0).all() and (want["dv"][1][0][:, weak] < 4e-3 * size[0]).all()
    for n in GRADIENTS:
        close(got[n], want[n], n)


@pytest.mark.parametrize("d", [64, 128])
def test_masked_buckets_beside_weak_keys(cuda_device, d):
    """A bias that masks every key behind the query, and keys with small weights."""
    x, valid, weak = weak_keys(d, 40, 57, seq=300, buckets=32)
    x["table"][:, 16:] = -np.inf
    c, got = run(x, valid, rb.Mask.FULL, 128)
    want = want_of(c)
    for n in GRADIENTS + ("dtable",):
        close(got[n], want[n], n)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in (c[:4] + (c[5].name(), c[6], c[7]))))
def test_tight_bounds_on_ordinary_inputs(cuda_device, case):
    batch, heads, seq, d, valid, mask, block, buckets, far = case
    x, valid = make(batch, heads, seq, d, valid, seq + d, buckets)
    c, got = run(x, valid, mask, block, max_distance=far or 128)
    want = want_of(c)
    for n in GRADIENTS + (("dtable",) if buckets else ()):
        close(got[n], want[n], n)


@pytest.mark.parametrize("d", [64, 96])
def test_rows_far_smaller_than_their_neighbours(cuda_device, d):
    """Operands that change by 2^20 from tile to tile, and by 2^12 within one."""
    x, valid = make(1, 2, 320, d, None, 58)
    at = np.arange(320)
    for n in ("v", "dout"):
        x[n] *= (2.0 ** (20 * (at // 64 % 2) - 10 - 12 * (at % 5 == 3)))[None, None, :, None].astype(np.float32)
    c, got = run(x, valid, rb.Mask.FULL, 128)
    want = want_of(c)
    for n in GRADIENTS:
        close(got[n], want[n], n)
