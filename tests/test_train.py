"""The training operators without a GPU: the bias's buckets, the workspace,
what the entry points refuse before any device work, and the plain form's
gradients against differences."""
import ctypes

import numpy as np
import pytest

import raya_b200 as rb
from raya_b200 import _lib
from _train import buckets_of, reference

LIB = _lib.lib


def bounds(buckets, max_distance):
    out = (ctypes.c_int32 * max(buckets // 2, 1))()
    st = LIB.raya_attn_bias_bounds(buckets, max_distance, out)
    return st, list(out)


@pytest.mark.parametrize("buckets,max_distance", [(4, 2), (4, 500), (6, 3), (8, 16), (16, 64), (32, 128), (32, 9),
                                                  (64, 256), (64, 512), (64, 4096), (64, 2 ** 29 - 1), (30, 128)])
def test_bucket_bounds_are_the_definition_in_whole_numbers(buckets, max_distance):
    st, got = bounds(buckets, max_distance)
    assert st == _lib.OK
    half, first = buckets // 2, buckets // 4
    rest = half - first
    for k in range(half):
        if k < first:
            assert got[k] == k
            continue
        want = first ** (rest - (k - first)) * max_distance ** (k - first)
        n = got[k]
        assert n ** rest >= want and (n == 0 or (n - 1) ** rest < want), (k, n)


def test_bucket_borders_that_floating_point_logs_miss():
    """first * ratio^(k / rest) is whole at every second bucket here."""
    assert bounds(32, 128)[1][8::2] == [8, 16, 32, 64]
    assert bounds(16, 64)[1][4:] == [4, 8, 16, 32]


@pytest.mark.parametrize("buckets,max_distance", [(32, 128), (4, 2), (30, 100)])
def test_python_buckets(buckets, max_distance):
    class Table:
        shape = (3, buckets)

    rel = np.arange(-700, 701)
    got = rb.RelativeBias(Table(), max_distance).bucket(rel)
    assert np.array_equal(got, buckets_of(rel, buckets, max_distance))
    assert got.min() == 0 and got.max() == buckets - 1


@pytest.mark.parametrize("buckets,max_distance,status", [(3, 128, 3), (2, 128, 3), (0, 128, 3), (-2, 128, 3), (66, 128, 3), (128, 128, 3),
                                                         (32, 8, 1), (32, 0, 1), (32, -5, 1), (32, 2 ** 29, 1)])
def test_bad_buckets_are_refused(buckets, max_distance, status):
    assert bounds(buckets, max_distance)[0] == status


def desc(batch=2, heads=3, seq=70, head_dim=64, mask=_lib.MASK_BLOCK, block=64, halo=1, window=0, scale=0.125):
    return _lib.Desc(batch, heads, seq, head_dim, block, mask, halo, window, scale)


BIAS = _lib.Bias(1024, 32, 128)


def forward(d, q=16, k=16, v=16, out=16, stats=16, bias=BIAS, ws=16, n=0):
    return LIB.raya_attn_forward_bias(d, q, k, v, out, stats, None, bias, ws, n, None)


def backward(d, q=16, k=16, v=16, out=16, stats=16, dout=16, dq=16, dk=16, dv=16, bias=BIAS, dtable=16, ws=16, n=0):
    return LIB.raya_attn_backward(d, q, k, v, out, stats, dout, dq, dk, dv, None, bias, dtable, ws, n, None)


def need(d, bias, back):
    n = ctypes.c_size_t()
    assert LIB.raya_attn_train_workspace(d, bias, back, ctypes.byref(n)) == _lib.OK, _lib.last_error()
    return n.value


@pytest.mark.parametrize("call,back", [(forward, 0), (backward, 1)])
def test_a_small_workspace_is_refused_with_its_length(call, back):
    d = desc()
    want = need(d, BIAS, back)
    assert want > 0
    for got in (0, want - 1):
        assert call(d, n=got) == _lib.ERR_LENGTH
        info = rb.last_error_info()
        assert (info.name, info.got, info.expected) == ("workspace", got, want)
    assert call(d, ws=None, n=want) == _lib.ERR_LENGTH
    assert call(d, ws=24, n=want) == _lib.ERR_UNSUPPORTED and "16-byte" in _lib.last_error()


def test_null_and_misaligned_tensors_are_refused():
    d, n = desc(), 1 << 40
    for name in ("q", "k", "v", "out"):
        assert forward(d, n=n, **{name: None}) == _lib.ERR_SHAPE and "null" in _lib.last_error()
        assert forward(d, n=n, **{name: 20}) == _lib.ERR_UNSUPPORTED and "16-byte" in _lib.last_error()
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        assert backward(d, n=n, **{name: None}) == _lib.ERR_SHAPE and "null" in _lib.last_error()
        assert backward(d, n=n, **{name: 24}) == _lib.ERR_UNSUPPORTED
    assert backward(d, n=n, stats=None) == _lib.ERR_SHAPE
    assert backward(d, n=n, stats=20) == _lib.ERR_UNSUPPORTED and "stats" in _lib.last_error()
    assert forward(d, n=n, stats=20) == _lib.ERR_UNSUPPORTED
    assert forward(d, n=n, bias=_lib.Bias(None, 32, 128)) == _lib.ERR_SHAPE and "table" in _lib.last_error()
    assert backward(d, n=n, bias=None) == _lib.ERR_SHAPE and "without a bias" in _lib.last_error()


def test_bad_shapes_and_biases_are_refused():
    n = 1 << 40
    for d, status in ((desc(head_dim=12), _lib.ERR_SHAPE), (desc(head_dim=264), _lib.ERR_UNSUPPORTED),
                      (desc(batch=0), _lib.ERR_SHAPE), (desc(heads=0), _lib.ERR_SHAPE), (desc(seq=-1), _lib.ERR_SHAPE),
                      (desc(block=0), _lib.ERR_UNSUPPORTED), (desc(halo=-1), _lib.ERR_SHAPE),
                      (desc(mask=7), _lib.ERR_UNSUPPORTED), (desc(mask=_lib.MASK_WINDOW, window=-1), _lib.ERR_SHAPE),
                      (desc(scale=float("nan")), _lib.ERR_SHAPE), (desc(seq=1 << 29), _lib.ERR_UNSUPPORTED),
                      (desc(batch=1 << 40), _lib.ERR_UNSUPPORTED), (desc(batch=1 << 62, heads=1 << 40), _lib.ERR_UNSUPPORTED),
                      (desc(batch=1 << 16, heads=1 << 12, seq=1 << 28), _lib.ERR_UNSUPPORTED)):
        assert forward(d, n=n) == status, _lib.last_error()
        assert backward(d, n=n) == status
        m = ctypes.c_size_t()
        assert LIB.raya_attn_train_workspace(d, None, 1, ctypes.byref(m)) == status
    for bias, status in ((_lib.Bias(1024, 31, 128), _lib.ERR_UNSUPPORTED), (_lib.Bias(1024, 66, 128), _lib.ERR_UNSUPPORTED),
                         (_lib.Bias(1024, 32, 4), _lib.ERR_SHAPE)):
        assert forward(desc(), bias=bias, n=n) == status
        assert backward(desc(), bias=bias, n=n) == status
    assert LIB.raya_attn_train_workspace(desc(), None, 1, None) == _lib.ERR_SHAPE
    assert LIB.raya_attn_bias_bounds(32, 128, None) == _lib.ERR_SHAPE
    assert forward(None, n=n) == _lib.ERR_SHAPE


def test_no_rows_is_no_work():
    """seq 0: nothing to write, no pointer looked at (without a bias gradient)."""
    assert forward(desc(seq=0), q=None, out=None, ws=None) == _lib.OK
    assert backward(desc(seq=0), q=None, dq=None, ws=None, bias=None, dtable=None) == _lib.OK
    assert need(desc(seq=0), BIAS, 1) == 0


def test_python_calls_take_cuda_tensors_only():
    import torch

    shape = rb.AttnShape(heads=1, seq=4, head_dim=64)
    params = rb.AttnParams.new(rb.Mask.FULL, 4, 64)
    x = torch.zeros(1, 1, 4, 64)
    with pytest.raises(TypeError, match="`q` must be a contiguous CUDA"):
        rb.Cuda().attend_bias(shape, params, x, x, x, x)
    with pytest.raises(TypeError, match="stats"):
        rb.Cuda().attend_backward(shape, params, x, x, x, x, None, x, x, x, x)
    assert rb.train_workspace(shape, params) == need(desc(1, 1, 4, 64, _lib.MASK_FULL), None, 0)
    assert rb.train_workspace(shape, params, backward=True) == need(desc(1, 1, 4, 64, _lib.MASK_FULL), None, 1)


@pytest.mark.parametrize("mask", [rb.Mask.block(1), rb.Mask.sliding(3), rb.Mask.FULL])
def test_reference_gradients_against_differences(mask):
    rng = np.random.default_rng(3)
    b, h, s, d, block = 2, 2, 9, 8, 4
    valid = np.array([9, 6])
    q, k, v, g = (rng.standard_normal((b, h, s, d)) for _ in range(4))
    table = rng.standard_normal((h, 8))
    at = {"q": q, "k": k, "v": v, "table": table}
    run = lambda: reference(mask, block, 0.4, valid, q, k, v, g, table, 6)  # noqa: E731
    got = run()
    loss = lambda: float((np.where(np.arange(s)[None, None, :, None] < valid[:, None, None, None], g, 0) * run()["out"][0]).sum())  # noqa: E731
    step = 1e-5
    for name in ("q", "k", "v", "table"):
        x, grad = at[name], got["d" + name][0]
        for _ in range(12):
            i = tuple(rng.integers(0, n) for n in x.shape)
            was = x[i]
            x[i] = was + step
            up = loss()
            x[i] = was - step
            down = loss()
            x[i] = was
            # the central difference is off by step^2 / 6 times a third derivative of order 10, and by rounding / step
            assert abs((up - down) / (2 * step) - grad[i]) < 1e-8 + 1e-9 * abs(grad[i]), (name, i)


@pytest.mark.parametrize("mask,buckets", [(rb.Mask.block(1), 8), (rb.Mask.sliding(30), 0), (rb.Mask.FULL, 8)])
def test_tight_bounds_have_the_references_values(mask, buckets):
    from _train_tight import small, tight

    rng = np.random.default_rng(4)
    valid = np.array([140, 77])
    q, k, v, g = (rng.standard_normal((2, 2, 140, 16)) for _ in range(4))
    k[:, :, 5] *= 30
    table = rng.standard_normal((2, buckets)) if buckets else None
    have, want = (f(mask, 32, 0.25, valid, q, k, v, g, table, 6) for f in (tight, reference))
    for n in want:
        assert np.array_equal(have[n][0], want[n][0]), n
        bound = np.broadcast_to(have[n][1], want[n][0].shape)
        assert np.isfinite(bound).all() and (bound >= 0).all(), n
    x = small(k)
    for r in range(140):
        assert (x[:, :, r, 0] == 2.0 ** -40 * np.abs(k[:, :, r // 64 * 64 : r // 64 * 64 + 64]).max((2, 3))).all()


@pytest.mark.parametrize("buckets,max_distance", [(32, 2 ** 32 + 128), (32, 2 ** 31), (32, -(2 ** 32) + 128), (32, 2 ** 64 + 128), (2 ** 32 + 32, 128)])
def test_sizes_beyond_32_bits_are_refused_in_python(buckets, max_distance):
    """The library takes 32-bit integers: what does not fit is refused, not cut to one that does."""
    class Table:
        shape = (3, buckets)

    bias = rb.RelativeBias(Table(), max_distance)
    shape, params = rb.AttnShape(heads=3, seq=70, head_dim=64), rb.AttnParams.new(rb.Mask.FULL, 70, 64)
    refused = rb.ShapeError if buckets == 32 else rb.UnsupportedError
    for call in (bias.bounds, lambda: bias.bucket(5), lambda: rb.train_workspace(shape, params, bias)):
        with pytest.raises(refused):
            call()


def test_sizes_may_be_numpy_integers():
    class Table:
        shape = (3, np.int64(32))

    assert np.array_equal(rb.RelativeBias(Table(), np.int64(128)).bounds(), bounds(32, 128)[1])
    with pytest.raises(TypeError):
        rb.RelativeBias(Table(), 128.5).bounds()
