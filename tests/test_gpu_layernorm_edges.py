"""Layer normalisation where other tests do not look: GeLU behind the norm, against float64 and against differences; rows whose sum
overflows; how optional arguments move the order of sums."""
import numpy as np
import pytest

import packed_oracle as po
from cases import rng_normal as Nrm
from test_gpu_layernorm import inputs, run_backward, run_forward, up, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    import mi355tensor
    mi355tensor.init(0)
    return mi355tensor


A, CUBE = float(np.sqrt(np.float32(2) / np.float32(3.141592654))), 0.044715


def gelu(v):
    return 0.5 * v * (1 + np.tanh(A * (v + CUBE * v ** 3)))


def gelu_slope(v):
    t = np.tanh(A * (v + CUBE * v ** 3))
    return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * A * (1 + 3 * CUBE * v * v)


def gelu_backward(delta, x, gamma, beta, mean, ivar):
    """As packed_oracle.backward, with the derivative of GeLU: error, dgamma, dbeta in float64 and what fp32 may add.  The slope's
    second derivative is at most 1; its own arithmetic: exp(-2u) is off by 3 + 5 * 2u half steps, and 2u * exp(-2u) <= 0.37, which makes 8 half
    steps of s and, with |2 v s (1 - s) u'| <= 0.6 and five products more, 15 to 25 of the slope: 32."""
    U = po.U
    rows, n, _ = po.row_view(x.shape, gamma.shape)
    f, dl, g, b, m, iv = (a.astype(np.float64).reshape(s) for a, s in ((x, (rows, n)), (delta, (rows, n)), (gamma, (1, n)), (beta, (1, n)), (mean, (rows, 1)), (ivar, (rows, 1))))
    xhat = (f - m) * iv
    pre = g * xhat + b
    front = dl * gelu_slope(pre)
    e_pre = 3 * U * np.abs(g * xhat) + U * np.abs(pre)
    e_front = np.abs(dl) * (e_pre + 32 * U) + U * np.abs(front)
    u = front * g
    e_u = np.abs(g) * e_front
    want = po.backward(front.reshape(x.shape), x, gamma, beta, mean, ivar, None)     # the rest of the pass, and the bounds of its own roundings
    e_c1, e_c2 = e_u.mean(1, keepdims=True), (e_u * np.abs(xhat)).mean(1, keepdims=True)
    want["error_tol"] += (iv * (e_u + e_c1 + np.abs(xhat) * e_c2)).reshape(x.shape) + U * np.abs(iv * u).reshape(x.shape)
    want["dgamma_tol"] += (e_front * np.abs(xhat)).sum(0).reshape(gamma.shape)
    want["dbeta_tol"] += e_front.sum(0).reshape(gamma.shape)
    return want


def test_the_slope_is_the_derivative():
    v, h = np.linspace(-8, 8, 4001), 1e-5
    assert np.abs(gelu_slope(v) - (gelu(v + h) - gelu(v - h)) / (2 * h)).max() < 1e-9
    assert np.abs(np.diff(gelu_slope(v)) / np.diff(v)).max() < 1


@pytest.mark.parametrize("n", [1, 33, 60, 1001, 2048, 10319, 20000, 40000])
def test_gelu(mt, n):
    x, gamma, beta, delta = inputs(n + 5, (4, 1, n, 1), (1, 1, n, 1))
    gamma *= 2                                                    # both tails
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, "gelu", packed=True)
    within(out, po.forward(x, gamma, beta, 1e-6, "gelu"), "out")
    for source, v in ((x, x), (pk, po.through_8_bits(x))):
        back = gelu_backward(delta, v, gamma, beta, mean, ivar)
        got, over = run_backward(mt, delta, source, gamma, beta, mean, ivar, "gelu"), run_backward(mt, delta, source, gamma, beta, mean, ivar, "gelu", inplace=True)
        for key, g in got.items():
            within(g, back, key)
            assert np.array_equal(g, over[key])


@pytest.mark.parametrize("rows,n", [(700, 64), (600, 1024), (520, 17001)])
def test_gelu_many_rows(mt, rows, n):
    x, gamma, beta, delta = inputs(rows + n, (rows, 1, n, 1), (1, 1, n, 1))
    _, mean, ivar, pk = run_forward(mt, x, gamma, beta, "gelu", packed=True)
    for source, v in ((x, x), (pk, po.through_8_bits(x))):
        back = gelu_backward(delta, v, gamma, beta, mean, ivar)
        for key, got in run_backward(mt, delta, source, gamma, beta, mean, ivar, "gelu").items():
            within(got, back, key)


def test_gelu_far_out(mt):
    """Slopes of 0 and 1 where the cube overflows, no NaN but of a NaN."""
    n = 64
    x = np.tile(np.float32([1, -1]), n // 2).reshape(1, 1, n, 1)
    gamma, beta = np.ones((1, 1, n, 1), np.float32), np.zeros((1, 1, n, 1), np.float32)
    gamma[0, 0, :, 0] = np.float32(10.0) ** (np.arange(n) % 38)
    mean, ivar = np.zeros((1, 1, 1, 1), np.float32), np.ones((1, 1, 1, 1), np.float32)
    got = run_backward(mt, np.ones((1, 1, n, 1), np.float32), x, gamma, beta, mean, ivar, "gelu")
    far = np.arange(n) % 38 >= 2
    assert np.array_equal(got["dbeta"].ravel()[far], (x.ravel() > 0).astype(np.float32)[far])
    beta[0, 0, 5, 0] = np.nan
    assert np.flatnonzero(np.isnan(run_backward(mt, np.ones((1, 1, n, 1), np.float32), x, gamma, beta, mean, ivar, "gelu")["dbeta"].ravel())).tolist() == [5]


@pytest.mark.parametrize("func", ["gelu", "sigmoid", "leaky_relu", "relu"])
@pytest.mark.parametrize("n", [50, 1000, 20000])
def test_gradients_against_differences(mt, n, func):
    """error, dgamma and dbeta against central differences of sum(delta * func(layernorm(..))) in float64 along random directions."""
    shape, pshape = (3, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n + 9, shape, pshape)
    _, mean, ivar, _ = run_forward(mt, x, gamma, beta, func)
    got = run_backward(mt, delta, x, gamma, beta, mean, ivar, func)
    f = gelu if func == "gelu" else lambda v: po.func(func, v)

    def pre(xv, gv, bv):
        d = xv - xv.mean((1, 2, 3), keepdims=True)
        return gv * d / np.sqrt((d * d).mean((1, 2, 3), keepdims=True) + float(np.float32(1e-6))) + bv

    at = [a.astype(np.float64) for a in (x, gamma, beta)]
    h = 1e-6
    for k, key in enumerate(("error", "dgamma", "dbeta")):
        direction = Nrm(k + 70, *at[k].shape).astype(np.float64)
        ends = [pre(*(a + sign * h * direction if i == k else a for i, a in enumerate(at))) for sign in (1, -1)]
        weight = delta.astype(np.float64)
        if func in ("relu", "leaky_relu"):
            # a value that changes its side, or stands within fp32's reach of zero, has two slopes: each such one may move the result by
            # its whole slope
            near = (np.sign(ends[0]) != np.sign(ends[1])) | (np.abs(ends[0]) < 1e-5)
        else:
            near = np.zeros(shape, bool)
        kinks = (np.abs(weight * (ends[0] - ends[1])) / (2 * h) * near).sum()
        slope, mine = ((f(ends[0]) - f(ends[1])) * weight).sum() / (2 * h), float((got[key].astype(np.float64) * direction).sum())
        # fp32: 6e-7 absolute in a slope (hardware exponential, 32 half steps of GeLU's 2e-6) times delta times the move of its value, at random
        # signs within four deviations; 1e-6 of the sum's size from rounding; differences: h^2 and 1e-16 * |loss| / h
        moves = np.linalg.norm(weight * (ends[0] - ends[1]) / (2 * h))
        slack = 4 * 2e-6 * moves + 1e-6 * np.abs(got[key] * direction).sum() + 1e-9 * np.abs(weight).sum()
        assert abs(slope - mine) <= slack + kinks, key


@pytest.mark.parametrize("n", [1024, 4096, 40000])
def test_a_sum_that_overflows(mt, n):
    """Finite values whose sum fp32 does not hold: NaN, in that row alone."""
    shape, pshape = (3, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n, shape, pshape)
    clean = run_forward(mt, x, gamma, beta)
    x[1] = 1e36
    out, mean, ivar, _ = run_forward(mt, x, gamma, beta)
    assert np.isnan(out[1]).all() and not np.isfinite(mean[1]).any() and np.array_equal(out[[0, 2]], clean[0][[0, 2]])
    assert np.isnan(run_backward(mt, delta, x, gamma, beta, mean, ivar)["error"][1]).all()


@pytest.mark.parametrize("n", [130, 333, 1001, 1023])
def test_the_8_bit_copy_beside_rows_of_odd_length(mt, n):
    """Such rows are summed in another order when the input is kept in 8 bits on the way: within the bounds both times."""
    x, gamma, beta, _ = inputs(n, (40, 1, n, 1), (1, 1, n, 1))
    want = po.forward(x, gamma, beta, 1e-6, "tangence")
    for packed in (False, True):
        for key, got in zip(("out", "mean", "ivar"), run_forward(mt, x, gamma, beta, "tangence", packed=packed)):
            within(got, want, key)


@pytest.mark.parametrize("n", [8193, 10319, 16384])
@pytest.mark.parametrize("func", [None, "sigmoid"])
def test_the_error_with_other_arguments(mt, n, func):
    """Rows of 8193 to 16384 values take other kernels with the number of rows and with the gradients that are wanted: the error of a row
    within its bounds whatever is asked for beside it."""
    rows = 1100
    x, gamma, beta, delta = inputs(n, (rows, 1, n, 1), (1, 1, n, 1))
    _, mean, ivar, pk = run_forward(mt, x, gamma, beta, func, packed=True)
    tg, tb = up(mt, gamma), up(mt, beta)
    for kept in (False, True):
        back = po.backward(delta, po.through_8_bits(x) if kept else x, gamma, beta, mean, ivar, func)
        for count in (rows, 600, 7):
            part = {key: back[key][:count] for key in ("error", "error_tol")}
            source = up(mt, x[:count])
            if kept:
                source = mt.CPackedTensor(count, 1, n, 1)
                mt.CTensorMath.Pack(source, up(mt, x[:count]))
            for wanted in (True, False):
                error = mt.CTensor(count, 1, n, 1)
                grads = (mt.CTensor(*gamma.shape), mt.CTensor(*gamma.shape)) if wanted else (None, None)
                mt.Fused.LayerNormBackward(error, *grads, up(mt, delta[:count]), tg, source, up(mt, mean[:count]), up(mt, ivar[:count]), beta=tb, func=func, accumulate=False)
                within(error.numpy(), part, "error")
