"""The linear layer's gradient from 8 bits where other tests do not look: what a ReLU leaves, features that are always 0, one sample that
outweighs the others."""
import numpy as np
import pytest

import packed_oracle as po
from cases import rng_normal as Nrm
from test_gpu_packed import run_linear, unequal

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


@pytest.fixture
def variant(mt, request):
    """The option that makes the call take one variant, whatever it would choose."""
    mt.set_option("linear_packed", request.param)
    yield request.param
    mt.set_option("linear_packed", 0)


KINDS, PARTS = (1, 2, 3, 4, 5), (1, 2, 3, 9)
VARIANTS = [k + 10 * s for k in KINDS for s in PARTS]


@pytest.mark.parametrize("variant", VARIANTS, indirect=True)
@pytest.mark.parametrize("b,n_in,n_out", [(1, 130, 6), (65, 257, 130), (200, 385, 66), (700, 129, 258), (333, 16, 33), (1300, 20, 2)])
def test_every_variant(mt, variant, b, n_in, n_out):
    """Against float64: normal activations, with a bias, added to what is there, the same bits again, in shifted memory."""
    x, delta = (Nrm(b, b, 1, n_in, 1) + 0.3).astype(np.float32), Nrm(b + 1, b, 1, n_out, 1, std=0.1)
    want, bound = bounds(delta.reshape(b, n_out), x)
    dw, db = run_linear(mt, x, delta)
    assert (np.abs(dw - want["dweight"]) <= bound).all() and (np.abs(db - want["dbias"]) <= want["dbias_tol"]).all()
    start = (Nrm(3, 1, 1, n_out, n_in), Nrm(4, 1, 1, n_out, 1))
    added = run_linear(mt, x, delta, accumulate=True, start=start)
    assert np.array_equal(added[0], start[0].reshape(n_out, n_in) + dw) and np.array_equal(added[1], start[1].ravel() + db)
    alone = run_linear(mt, x, delta, bias=False)
    assert np.array_equal(alone[0], dw) and (alone[1] == 7).all()
    pk, shifted = mt.CPackedTensor(*x.shape), []
    mt.CTensorMath.Pack(pk, mt.CTensor.from_numpy(x))
    for a, shape in ((delta, delta.shape), (None, (1, 1, n_out, n_in)), (None, (1, 1, n_out, 1))):
        n = int(np.prod(shape))
        whole = mt.CTensor.from_numpy(np.concatenate([[9], np.full(n, 7) if a is None else a.ravel(), np.full(8, 9)]).astype(np.float32).reshape(1, 1, 1, -1))
        shifted.append((whole, mt.CTensor.wrap(whole.ptr.value + 4, shape), n))
    mt.Fused.LinearBackwardWeightsSum(shifted[1][1], shifted[2][1], pk, shifted[0][1], accumulate=False)
    for (whole, _, n), w in zip(shifted[1:], (dw, db)):
        got = whole.numpy().ravel()
        assert np.array_equal(got[1:1 + n], w.ravel()) and got[0] == 9 and (got[1 + n:] == 9).all()


@pytest.mark.parametrize("variant", VARIANTS, indirect=True)
@pytest.mark.parametrize("what", ["samples without delta", "samples with little delta", "one feature's activations", "every row", "every sample", "rows of zeros",
                                  "one sample of a row", "constant activations"])
def test_every_variant_with_unequal_magnitudes(mt, variant, what):
    b, n_in, n_out = 700, 300, 260
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1, std=0.02)
    unequal(x, delta, what)
    dw, db = run_linear(mt, x, delta)
    want, bound = bounds(delta.reshape(b, n_out), x)
    assert (np.abs(dw - want["dweight"]) <= bound + 1e-44).all() and (np.abs(db - want["dbias"]) <= want["dbias_tol"] + 1e-44).all()


@pytest.mark.parametrize("variant", VARIANTS, indirect=True)
def test_every_variant_behind_a_relu(mt, variant):
    b, n_in, n_out = 650, 520, 130
    x, dead = relu_input(5, b, n_in)
    delta = Nrm(6, b, 1, n_out, 1, std=0.02)
    dw, _ = run_linear(mt, x, delta)
    want, bound = bounds(delta.reshape(b, n_out), x)
    assert (np.abs(dw - want["dweight"]) <= bound).all() and not dw[:, dead].any() and dw.any(0).sum() == n_in - dead.size


@pytest.mark.parametrize("variant", VARIANTS, indirect=True)
def test_every_variant_with_values_that_are_not_finite(mt, variant):
    b, n_in, n_out = 650, 300, 140
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1)
    fine = run_linear(mt, x, delta)
    bad = delta.copy()
    bad[b - 1, 0, 5, 0], bad[0, 0, 7, 0] = np.inf, np.nan
    dw, db = run_linear(mt, x, bad)
    assert np.isnan(dw[[5, 7]]).all() and np.isinf(db[5]) and np.isnan(db[7])
    others = [o for o in range(n_out) if o not in (5, 7)]
    assert np.array_equal(dw[others], fine[0][others]) and np.array_equal(db[others], fine[1][others])
    x[b - 1, 0, 129, 0] = np.nan
    dw, db = run_linear(mt, x, delta)
    assert np.isnan(dw[:, 128:256]).all() and np.array_equal(np.delete(dw, np.r_[128:256], 1), np.delete(fine[0], np.r_[128:256], 1)) and np.array_equal(db, fine[1])


@pytest.mark.parametrize("variant", [1, 2, 3, 4, 5], indirect=True)
def test_one_product(mt, variant):
    """A batch of one: every weight is one product.  Its roundings: delta * step (2^-24 of it, or 2^-23 in two fp16 numbers, whose smallest
    part is 2^-26 of the largest of its row), the sum of its parts on the matrix cores, low + zero * step and its product with delta, and the sum
    of both.  The first part times a whole number of 8 bits is exact (16 or 19 bits).  The second part of three is the upper 8 bits of what
    the first leaves, which may begin with zeros: with k of them the sum of two parts times 8 bits has 24 + k bits and is rounded, and so
    is the sum with the third.  So each part after the first adds one rounding."""
    n_in, n_out = 128, 2000
    x, delta = Nrm(1, 1, 1, n_in, 1), Nrm(2, 1, 1, n_out, 1)
    dw, _ = run_linear(mt, x, delta)
    q, low, step = po.pack(x)
    st, lo = float(step[0, 0]), float(low[0, 0])
    zero = np.clip(np.rint(-lo / st), 0, 255)
    d = delta.reshape(-1, 1).astype(np.float64)
    product, rest = d * st * (q.astype(np.float64) - zero), d * (lo + zero * st)
    share, parts = (2.0 ** -24, 2) if variant <= 3 else (2.0 ** -23 + 2.0 ** -26, 1)      # parts after the first
    assert (np.abs(dw - (product + rest)) <= (share + parts * po.U) * np.abs(product) + 2 * po.U * np.abs(rest) + po.U * 1.001 * np.abs(product + rest)).all()


def test_the_option_takes_the_variants_that_there_are(mt):
    for value in (-1, 6, 10, 17, 1 + 10 * 129):
        with pytest.raises(mt.TensorError) as e:
            mt.set_option("linear_packed", value)
        assert e.value.code == 6
    mt.set_option("linear_packed", 5 + 10 * 128)
    mt.set_option("linear_packed", 0)


# sizes at which the estimate takes a variant that no other test's size takes: 256 rows in three numbers; 256 rows in two, in parts; two groups of wavefronts
# in parts, in three and in two numbers
@pytest.mark.parametrize("b,n_in,n_out", [(361, 1333, 3302), (4163, 1792, 2712), (4685, 4248, 66), (4294, 5727, 40)])
def test_sizes_of_rare_variants(mt, b, n_in, n_out):
    x, delta = (Nrm(b, b, 1, n_in, 1) + 0.5).astype(np.float32), Nrm(b + 1, b, 1, n_out, 1, std=0.1)
    dw, db = run_linear(mt, x, delta)
    want, bound = bounds(delta.reshape(b, n_out), x)
    assert (np.abs(dw - want["dweight"]) <= bound).all() and (np.abs(db - want["dbias"]) <= want["dbias_tol"]).all()
