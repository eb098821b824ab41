"""The linear layer's gradient from 8 bits where other tests do not look: what a ReLU leaves, features that are always 0, one sample that
outweighs the others."""
import numpy as np
import pytest

import packed_oracle as po
from cases import rng_normal as Nrm
from test_gpu_packed import run_linear

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    import mi355tensor
    mi355tensor.init(0)
    return mi355tensor


def relu_input(seed, b, n_in):
    """Activations behind a ReLU, every seventh feature 0 in all samples, and a whole group of them where there is one."""
    x = np.maximum(Nrm(seed, b, 1, n_in, 1), 0)
    x[:, :, ::7] = 0
    if n_in >= 384:
        x[:, :, 128:256] = 0
    return x, np.flatnonzero(~x.any((0, 1, 3)))


def bounds(delta, x):
    """(gradient in float64, bound of every weight).  fp32 additions of at most B + 18 terms of the values' size; delta * step off by 2^-23
    of itself or 2^-26 of the largest of its row and group, times at most 255 steps."""
    want = po.linear_weights(delta, x)
    q, low, step = po.pack(x)
    largest = np.stack([(np.abs(delta.astype(np.float64)) * s[:, None]).max(0) for s in step.T.astype(np.float64)], 1)       # [Out,groups]
    per = np.repeat(np.arange(low.shape[1]), po.GROUP)[:q.shape[1]]
    # the steps between a value and 0 (or the end of its group's range nearest to 0)
    with np.errstate(all="ignore"):
        zero = np.clip(np.nan_to_num(-low.astype(np.float64) / step, nan=0.0, posinf=255, neginf=0), 0, 255)
    steps = np.abs(q - zero[:, per]) + 1
    steps[(q == 0) & (low[:, per] == 0)] = 0
    return want, want["dweight_tol"] + 2.0 ** -26 * largest[:, per] * steps.sum(0)


@pytest.mark.parametrize("b,n_in,n_out", [(1, 130, 5), (64, 300, 130), (512, 1024, 256), (3000, 1000, 100), (20000, 64, 48), (1500, 2000, 1500), (5000, 1000, 1501), (1100, 4000, 4000)])
def test_features_that_are_always_zero(mt, b, n_in, n_out):
    x, dead = relu_input(b, b, n_in)
    delta = Nrm(b + 1, b, 1, n_out, 1, std=0.02)
    dw, _ = run_linear(mt, x, delta)
    assert dead.size and not dw[:, dead].any()
    start = (Nrm(3, 1, 1, n_out, n_in), np.zeros((1, 1, n_out, 1), np.float32))
    added, _ = run_linear(mt, x, delta, accumulate=True, start=start)
    assert np.array_equal(added[:, dead], start[0].reshape(n_out, n_in)[:, dead])


@pytest.mark.parametrize("b,n_in,n_out", [(64, 300, 130), (512, 130, 64), (1500, 2000, 300), (3000, 257, 1000)])
@pytest.mark.parametrize("what", ["relu", "leaky relu", "normal", "below zero", "far from zero"])
@pytest.mark.parametrize("outlier", [1, 1e5])
def test_the_sums_are_of_the_size_of_the_values(mt, b, n_in, n_out, what, outlier):
    x = relu_input(b, b, n_in)[0] if what == "relu" else Nrm(b, b, 1, n_in, 1)
    if what == "leaky relu":
        x = np.where(x > 0, x, np.float32(0.01) * x)
    elif what == "below zero":
        x = -np.abs(x)
    elif what == "far from zero":
        x = x + np.float32(100)
    delta = Nrm(b + 1, b, 1, n_out, 1, std=0.02)
    delta[b // 2] *= np.float32(outlier)
    dw, _ = run_linear(mt, x, delta)
    want, bound = bounds(delta.reshape(b, n_out), x)
    off = np.abs(dw - want["dweight"])
    assert (off <= bound).all(), float((off / (bound + 1e-44)).max())
