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
