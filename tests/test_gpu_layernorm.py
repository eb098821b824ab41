"""Layer normalisation on the GPU against float64, with the bounds that fp32 arithmetic allows (packed_oracle.py)."""
import ctypes as C

import numpy as np
import pytest

import packed_oracle as po
from cases import rng_normal as Nrm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt():
    import mi355tensor
    mi355tensor.init(0)
    return mi355tensor


def up(mt, a, shift=0):
    """On the device; `shift` floats behind a 16-byte boundary."""
    a = np.ascontiguousarray(a, np.float32)
    if not shift:
        return mt.CTensor.from_numpy(a)
    whole = mt.CTensor.from_numpy(np.concatenate([np.full(shift, np.nan, np.float32), a.ravel(), np.full(4, np.nan, np.float32)]).reshape(1, 1, 1, -1))
    t = mt.CTensor.wrap(whole.ptr.value + 4 * shift, a.shape)
    t._base = whole
    return t


def inputs(seed, shape, pshape, offset=0.7, scale=1.5):
    x = Nrm(seed, *shape) * scale + offset + Nrm(seed + 1, *pshape)
    return x.astype(np.float32), (1 + 0.3 * Nrm(seed + 2, *pshape)).astype(np.float32), (0.2 * Nrm(seed + 3, *pshape)).astype(np.float32), Nrm(seed + 4, *shape, std=0.1)


def within(got, want, key):
    off = np.abs(np.asarray(got, np.float64) - want[key])
    bad = ~(off <= want[key + "_tol"] + 1e-44)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of the bound" % (key, bad.sum(), bad.size, np.max(off / (want[key + "_tol"] + 1e-44)))


def run_forward(mt, x, gamma, beta, func=None, eps=1e-6, packed=False, shift=0, inplace=False):
    _, _, stat = po.row_view(x.shape, gamma.shape)
    tx, out = up(mt, x, shift), up(mt, np.full(x.shape, 7, np.float32), shift)
    mean, ivar = up(mt, np.full(stat, 7, np.float32)), up(mt, np.full(stat, 7, np.float32))
    pk = mt.CPackedTensor(*x.shape) if packed else None
    mt.Fused.LayerNormForward(tx if inplace else out, tx, up(mt, gamma, shift), up(mt, beta, shift), mean, ivar, pk, eps, func)
    return (tx if inplace else out).numpy(), mean.numpy(), ivar.numpy(), pk


def run_backward(mt, delta, x, gamma, beta, mean, ivar, func=None, shift=0, accumulate=False, start=None, inplace=False):
    """x: an array, or a packed tensor on the device."""
    td, error = up(mt, delta, shift), up(mt, np.full(delta.shape, 7, np.float32), shift)
    dg, db = (up(mt, np.full(gamma.shape, 7, np.float32) if start is None else s, shift) for s in (start or (0, 0)))
    mt.Fused.LayerNormBackward(td if inplace else error, dg, db, td, up(mt, gamma, shift), x if isinstance(x, mt.CPackedTensor) else up(mt, x, shift), up(mt, mean),
                               up(mt, ivar), beta=up(mt, beta, shift), func=func, accumulate=accumulate)
    return {"error": (td if inplace else error).numpy(), "dgamma": dg.numpy(), "dbeta": db.numpy()}


# rows of every length at which a kernel, a vector width, a group or a split of a row can change
ROWS = [1, 2, 3, 4, 7, 16, 31, 32, 33, 64, 65, 100, 127, 128, 129, 132, 255, 256, 257, 260, 500, 511, 512, 513, 516, 777, 1000, 1023, 1024, 1025, 1028, 1920, 2047, 2048,
        2049, 2052, 3000, 4095, 4096, 4097, 4100, 6144, 8191, 8192, 8193, 8196, 10000, 12345, 16383, 16384, 16385, 16388, 20000, 32767, 32768, 32769, 32772, 40000,
        65536, 65537, 100001, 147456, 200003]


@pytest.mark.parametrize("n", ROWS)
def test_row_lengths(mt, n):
    count = 5 if n <= 20000 else 3
    shape, pshape = (count, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n, shape, pshape)
    want = po.forward(x, gamma, beta, 1e-6, None)
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, packed=True)
    for key, got in (("out", out), ("mean", mean), ("ivar", ivar)):
        within(got, want, key)
    # the 8 bits that the forward pass leaves are those of mt_pack
    values = mt.CTensor(*shape)
    mt.CTensorMath.Unpack(values, pk)
    kept = po.through_8_bits(x)
    assert np.array_equal(values.numpy(), kept)
    for source, v in ((x, x), (pk, kept)):
        back = po.backward(delta, v, gamma, beta, mean, ivar, None)
        for key, got in run_backward(mt, delta, source, gamma, beta, mean, ivar).items():
            within(got, back, key)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 31, 63, 64, 65, 255, 257, 1000, 4099])
@pytest.mark.parametrize("n", [24, 130, 1000, 1024])
def test_row_counts(mt, rows, n):
    x, gamma, beta, delta = inputs(rows * 7 + n, (rows, 1, n, 1), (1, 1, n, 1))
    want = po.forward(x, gamma, beta, 1e-5, None)
    out, mean, ivar, _ = run_forward(mt, x, gamma, beta, eps=1e-5)
    for key, got in (("out", out), ("mean", mean), ("ivar", ivar)):
        within(got, want, key)
    back = po.backward(delta, x, gamma, beta, mean, ivar, None)
    for key, got in run_backward(mt, delta, x, gamma, beta, mean, ivar).items():
        within(got, back, key)


# what a row spans, with sizes at which groups of 128 straddle rows and planes
GEOMETRIES = [((3, 4, 5, 6), (1, 4, 5, 6)), ((3, 4, 5, 6), (1, 1, 5, 6)), ((3, 4, 5, 6), (1, 1, 1, 6)), ((2, 3, 48, 64), (1, 3, 48, 64)), ((2, 16, 24, 32), (1, 1, 24, 32)),
              ((7, 1, 5, 1000), (1, 1, 1, 1000)), ((5, 2, 3, 128), (1, 1, 1, 128)), ((4, 3, 1, 96), (1, 1, 1, 96)), ((300, 1, 1, 10), (1, 1, 1, 10)),
              ((2, 3, 192, 256), (1, 3, 192, 256)), ((6, 2, 130, 130), (1, 1, 130, 130)), ((3, 2, 2, 9000), (1, 1, 1, 9000)), ((2, 2, 2, 33000), (1, 1, 1, 33000)),
              ((9, 3, 256, 1), (1, 1, 256, 1)), ((3, 5, 1, 256), (1, 1, 1, 256)), ((40, 3, 7, 11), (1, 3, 7, 11))]


@pytest.mark.parametrize("shape,pshape", GEOMETRIES)
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("func", [None, "sigmoid"])
def test_geometries(mt, shape, pshape, shift, func):
    x, gamma, beta, delta = inputs(sum(shape), shape, pshape)
    want = po.forward(x, gamma, beta, 1e-6, func)
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, func, packed=True, shift=shift)
    for key, got in (("out", out), ("mean", mean), ("ivar", ivar)):
        within(got, want, key)
    values = mt.CTensor(*shape)
    mt.CTensorMath.Unpack(values, pk)
    kept = po.through_8_bits(x)
    assert np.array_equal(values.numpy(), kept)
    for source, v in ((x, x), (pk, kept)):
        back = po.backward(delta, v, gamma, beta, mean, ivar, func)
        for key, got in run_backward(mt, delta, source, gamma, beta, mean, ivar, func, shift=shift).items():
            within(got, back, key)


@pytest.mark.parametrize("rows,n,func", [(600, 8196, "tangence"), (257, 16388, None), (530, 8195, "sigmoid"), (17, 16385, None), (300, 20000, "relu"), (16, 49152, None),
                                         (33, 49156, "tangence"), (520, 17001, None), (1030, 9001, None), (1024, 12291, None), (513, 12290, "sigmoid"),
                                         (20, 36866, None), (9, 36867, "tangence"), (1027, 16383, None)])
def test_many_long_rows(mt, rows, n, func):
    """Sums over rows that are cut into pieces: several groups of rows, groups of every size, error beside and over delta."""
    x, gamma, beta, delta = inputs(rows + n, (rows, 1, n, 1), (1, 1, n, 1))
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, func, packed=True)
    within(out, po.forward(x, gamma, beta, 1e-6, func), "out")
    for source, v in ((x, x), (pk, po.through_8_bits(x))):
        back = po.backward(delta, v, gamma, beta, mean, ivar, func)
        a, b = run_backward(mt, delta, source, gamma, beta, mean, ivar, func), run_backward(mt, delta, source, gamma, beta, mean, ivar, func, inplace=True)
        for key, got in a.items():
            within(got, back, key)
            assert np.array_equal(got, b[key])


@pytest.mark.parametrize("rows,n", [(5, 24), (700, 24), (600, 128), (9, 1024), (600, 1024), (5, 4096), (513, 4096), (7, 8192), (3, 16384), (600, 8192), (3, 32768), (20, 40000)])
@pytest.mark.parametrize("func", [None, "tangence"])
def test_past_the_caches(mt, rows, n, func):
    """What tensors of 128 MiB and more get, on small ones: the same bits, in place too where there are many rows."""
    x, gamma, beta, delta = inputs(rows + n, (rows, 1, n, 1), (1, 1, n, 1))
    results = []
    for option in (0, 1):
        mt.set_option("nontemporal", option)
        try:
            out, mean, ivar, pk = run_forward(mt, x, gamma, beta, func, packed=True)
            values = mt.CTensor(*x.shape)
            mt.CTensorMath.Unpack(values, pk)
            results.append([out, mean, ivar, values.numpy()])
            for source in (x, pk):
                for inplace in (False, True):
                    results[-1] += run_backward(mt, delta, source, gamma, beta, mean, ivar, func, inplace=inplace).values()
        finally:
            mt.set_option("nontemporal", 2)
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    assert all(np.array_equal(results[0][k], results[0][k + 3]) for k in (4, 5, 6, 10, 11, 12))


@pytest.mark.parametrize("packed", [False, True])
def test_long_rows_beyond_the_caches(mt, packed):
    """Rows in pieces, more of them than the caches hold: some at a time.  Every row as it would be alone."""
    n, rows = 40001, 2000
    x = mt.CTensor(rows, 1, n, 1)
    mt.CTensorMath.SetNormalNoise(x, 3)
    gamma, beta = up(mt, Nrm(1, 1, 1, n, 1)), up(mt, Nrm(2, 1, 1, n, 1))
    out, mean, ivar, pk = mt.CTensor(rows, 1, n, 1), mt.CTensor(rows, 1, 1, 1), mt.CTensor(rows, 1, 1, 1), mt.CPackedTensor(rows, 1, n, 1) if packed else None
    mt.Fused.LayerNormForward(out, x, gamma, beta, mean, ivar, pk, 1e-6, "tangence")
    m, v = mean.numpy().ravel(), ivar.numpy().ravel()
    values = mt.CTensor(rows, 1, n, 1)
    if packed:
        mt.CTensorMath.Unpack(values, pk)
    for row in (0, 1, 1046, 1047, 1048, 1049, 1999):   # around the rows at which a part of 160 MiB ends
        one = mt.CTensor.wrap(x.ptr.value + 4 * n * row, (1, 1, n, 1))
        o1, m1, v1, p1 = mt.CTensor(1, 1, n, 1), mt.CTensor(1, 1, 1, 1), mt.CTensor(1, 1, 1, 1), mt.CPackedTensor(1, 1, n, 1)
        mt.Fused.LayerNormForward(o1, one, gamma, beta, m1, v1, p1 if packed else None, 1e-6, "tangence")
        assert np.array_equal(mt.CTensor.wrap(out.ptr.value + 4 * n * row, (1, 1, n, 1)).numpy(), o1.numpy())
        assert m[row] == m1.numpy().item() and v[row] == v1.numpy().item()
        if packed:
            mt.CTensorMath.Unpack(o1, p1)
            assert np.array_equal(mt.CTensor.wrap(values.ptr.value + 4 * n * row, (1, 1, n, 1)).numpy(), o1.numpy())


def test_squares_that_overflow(mt):
    """Deviations above 1.8e19: no variance that fp32 holds, the row counts as having none of its values apart."""
    for n in (100, 1024, 4096, 40000):
        x = np.tile(np.float32([3e19, -3e19]), n // 2).reshape(1, 1, n, 1)
        gamma, beta = np.full((1, 1, n, 1), 2, np.float32), np.full((1, 1, n, 1), 0.25, np.float32)
        out, mean, ivar, _ = run_forward(mt, x, gamma, beta)
        assert (out == 0.25).all() and mean.item() == 0 and ivar.item() == 0


@pytest.mark.parametrize("func", ["sigmoid", "relu", "gelu", "leaky_relu", "linear", "tangence"])
@pytest.mark.parametrize("n", [60, 1001, 2048, 20000, 40000])
def test_functions(mt, func, n):
    x, gamma, beta, delta = inputs(n + 5, (4, 1, n, 1), (1, 1, n, 1))
    want = po.forward(x, gamma, beta, 1e-6, func)
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, func, packed=True)
    within(out, want, "out")
    for source, v in ((x, x), (pk, po.through_8_bits(x))):
        back = po.backward(delta, v, gamma, beta, mean, ivar, func)
        for key, got in run_backward(mt, delta, source, gamma, beta, mean, ivar, func).items():
            within(got, back, key)


@pytest.mark.parametrize("n", [50, 1000, 4096, 20000, 40000])
def test_gradients_against_differences(mt, n):
    """error, dgamma and dbeta against central differences of sum(delta * layernorm(..)) in float64 along random directions."""
    shape, pshape = (3, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n + 9, shape, pshape)
    _, mean, ivar, _ = run_forward(mt, x, gamma, beta, "tangence")
    got = run_backward(mt, delta, x, gamma, beta, mean, ivar, "tangence")

    def loss(xv, gv, bv):
        d = xv - xv.mean((1, 2, 3), keepdims=True)
        xhat = d / np.sqrt((d * d).mean((1, 2, 3), keepdims=True) + float(np.float32(1e-6)))
        return float((delta.astype(np.float64) * np.tanh(gv * xhat + bv)).sum())

    at = [a.astype(np.float64) for a in (x, gamma, beta)]
    h = 1e-5
    for k, key in enumerate(("error", "dgamma", "dbeta")):
        direction = Nrm(k + 70, *at[k].shape).astype(np.float64)
        ends = []
        for sign in (1, -1):
            moved = list(at)
            moved[k] = at[k] + sign * h * direction
            ends.append(loss(*moved))
        slope, mine = (ends[0] - ends[1]) / (2 * h), float((got[key].astype(np.float64) * direction).sum())
        # fp32: 3e-7 per element of a random sum from the fast tanh, 1e-6 of its size from rounding; differences: h^2 times the third
        # derivative (below 10 times the size) and 1e-16 * |loss| / h
        size = np.linalg.norm(got[key].astype(np.float64) * direction)
        noise = 6e-7 * np.linalg.norm(np.asarray(delta, np.float64)) * 4 * np.sqrt(3)
        assert abs(slope - mine) <= 1e-6 * np.abs(got[key] * direction).sum() + noise + 1e-9 * size + 1e-10 * np.abs(delta).sum(), key


@pytest.mark.parametrize("shape,pshape", [((6, 1, 50, 1), (1, 1, 50, 1)), ((6, 1, 1024, 1), (1, 1, 1024, 1)), ((6, 1, 4000, 1), (1, 1, 4000, 1)), ((3, 1, 40000, 1), (1, 1, 40000, 1)),
                                          ((700, 1, 64, 1), (1, 1, 64, 1))])
def test_gradients_add_to_what_is_there(mt, shape, pshape):
    x, gamma, beta, delta = inputs(31, shape, pshape)
    _, mean, ivar, pk = run_forward(mt, x, gamma, beta, packed=True)
    start = (Nrm(77, *pshape), Nrm(78, *pshape))
    for source in (x, pk):
        fresh = run_backward(mt, delta, source, gamma, beta, mean, ivar)
        added = run_backward(mt, delta, source, gamma, beta, mean, ivar, accumulate=True, start=start)
        assert np.array_equal(added["error"], fresh["error"])
        assert np.array_equal(added["dgamma"], start[0] + fresh["dgamma"]) and np.array_equal(added["dbeta"], start[1] + fresh["dbeta"])


@pytest.mark.parametrize("n", [10, 130, 1000, 1024, 4096, 9000, 20000, 40000])
def test_written_in_place(mt, n):
    """output over the input, error over delta: the same bits."""
    x, gamma, beta, delta = inputs(n, (9, 1, n, 1), (1, 1, n, 1))
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, "tangence", packed=True)
    again, mean2, ivar2, pk2 = run_forward(mt, x, gamma, beta, "tangence", packed=True, inplace=True)
    assert np.array_equal(out, again) and np.array_equal(mean, mean2) and np.array_equal(ivar, ivar2)
    for source, source2 in ((x, x), (pk, pk2)):
        a = run_backward(mt, delta, source, gamma, beta, mean, ivar, "tangence")
        b = run_backward(mt, delta, source2, gamma, beta, mean, ivar, "tangence", inplace=True)
        assert all(np.array_equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("n", [20, 1000, 1024, 4096, 20000, 40000])
def test_optional_results(mt, n):
    x, gamma, beta, delta = inputs(n, (5, 1, n, 1), (1, 1, n, 1))
    out, mean, ivar, _ = run_forward(mt, x, gamma, beta)
    o = mt.CTensor(*x.shape)
    mt.Fused.LayerNormForward(o, up(mt, x), up(mt, gamma), up(mt, beta))
    assert np.array_equal(o.numpy(), out)
    full = run_backward(mt, delta, x, gamma, beta, mean, ivar)
    for wanted in ("dgamma", "dbeta", None):
        e, g = mt.CTensor(*x.shape), mt.CTensor(*gamma.shape)
        mt.Fused.LayerNormBackward(e, g if wanted == "dgamma" else None, g if wanted == "dbeta" else None, up(mt, delta), up(mt, gamma), up(mt, x), up(mt, mean), up(mt, ivar),
                                   accumulate=False)
        assert np.array_equal(e.numpy(), full["error"])
        assert wanted is None or np.array_equal(g.numpy(), full[wanted])


@pytest.mark.parametrize("n", [1, 40, 1000, 4096, 20000, 40000])
@pytest.mark.parametrize("offset,scale", [(0.0, 0.0), (3.0, 0.0), (1e4, 1.0), (0.0, 1e-12), (0.0, 1e15)])
def test_constant_rows_large_offsets_and_scales(mt, n, offset, scale):
    x = (offset + scale * Nrm(n, 4, 1, n, 1)).astype(np.float32)
    gamma, beta, delta = np.ones((1, 1, n, 1), np.float32), np.full((1, 1, n, 1), 0.25, np.float32), Nrm(3, 4, 1, n, 1)
    want = po.forward(x, gamma, beta, 1e-6, None)
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, packed=True)
    for key, got in (("out", out), ("mean", mean), ("ivar", ivar)):
        within(got, want, key)
    for source, v in ((x, x), (pk, po.through_8_bits(x))):
        back = po.backward(delta, v, gamma, beta, mean, ivar, None)
        for key, got in run_backward(mt, delta, source, gamma, beta, mean, ivar).items():
            within(got, back, key)


@pytest.mark.parametrize("n", [12, 60, 1000, 1024, 4096, 20000, 40000])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_row_that_is_not_finite_stays_alone(mt, n, value):
    shape, pshape = (6, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n, shape, pshape)
    clean, mean0, ivar0, _ = run_forward(mt, x, gamma, beta)
    fine = run_backward(mt, delta, x, gamma, beta, mean0, ivar0)
    x[2, 0, n // 2, 0] = value
    out, mean, ivar, pk = run_forward(mt, x, gamma, beta, packed=True)
    others = [0, 1, 3, 4, 5]
    assert np.isnan(out[2]).all() and np.array_equal(out[others], clean[others]) and np.array_equal(mean[others], mean0[others])
    for source in (x, pk):
        got = run_backward(mt, delta, source, gamma, beta, mean, ivar)
        assert np.isnan(got["error"][2]).all() and np.isnan(got["dgamma"]).all() and np.isfinite(got["dbeta"]).all()
        if source is x:
            assert np.array_equal(got["error"][others], fine["error"][others])
            assert np.array_equal(got["dbeta"], fine["dbeta"])


def test_nothing_to_normalise(mt):
    for shape, pshape in (((0, 1, 8, 1), (1, 1, 8, 1)), ((3, 0, 4, 4), (1, 1, 4, 4)), ((3, 1, 0, 1), (1, 1, 0, 1))):
        x = np.zeros(shape, np.float32)
        gamma = np.ones(pshape, np.float32)
        out, mean, ivar, pk = run_forward(mt, x, gamma, gamma, packed=True)
        assert out.size == 0
        start = (np.full(pshape, 2, np.float32), np.full(pshape, 3, np.float32))
        for source in (x, pk):
            kept = run_backward(mt, x, source, gamma, gamma, mean, ivar, accumulate=True, start=start)
            assert np.array_equal(kept["dgamma"], start[0]) and np.array_equal(kept["dbeta"], start[1])
            none = run_backward(mt, x, source, gamma, gamma, mean, ivar)
            assert not none["dgamma"].any() and not none["dbeta"].any()


@pytest.mark.parametrize("rows,n", [(7, 100), (300, 1000), (100, 4096), (3, 50000)])
def test_same_bits_every_time(mt, rows, n):
    x, gamma, beta, delta = inputs(5, (rows, 1, n, 1), (1, 1, n, 1))
    first = run_forward(mt, x, gamma, beta, packed=True)
    back = [run_backward(mt, delta, s, gamma, beta, first[1], first[2]) for s in (x, first[3])]
    for _ in range(3):
        again = run_forward(mt, x, gamma, beta, packed=True)
        assert all(np.array_equal(a, b) for a, b in zip(first[:3], again[:3]))
        for s, b in zip((x, again[3]), back):
            got = run_backward(mt, delta, s, gamma, beta, first[1], first[2])
            assert all(np.array_equal(got[k], b[k]) for k in b)


@pytest.mark.parametrize("n", [30, 333, 1000, 1025, 1026, 1027, 4096, 5003, 9001, 36866, 36867, 40000])
def test_nothing_is_written_beside_the_results(mt, n):
    """Guard values in front of and behind every result stay."""
    shape, pshape = (5, 1, n, 1), (1, 1, n, 1)
    x, gamma, beta, delta = inputs(n, shape, pshape)

    def guarded(s):
        c = int(np.prod(s))
        whole = mt.CTensor.from_numpy(np.full((1, 1, 1, c + 128), 5, np.float32))
        t = mt.CTensor.wrap(whole.ptr.value + 256, s)
        t._base = whole
        return t

    def intact(t):
        a = t._base.numpy().ravel()
        return (a[:64] == 5).all() and (a[64 + t.count:] == 5).all()

    stat = (5, 1, 1, 1)
    out, mean, ivar, error, dg, db = (guarded(s) for s in (shape, stat, stat, shape, pshape, pshape))
    size = mt.CPackedTensor.bytes_of(shape)
    memory = mt.CTensor.from_numpy(np.full((1, 1, 1, size // 4 + 64), 5, np.float32))
    pk = mt.CPackedTensor.wrap(memory.ptr.value + 128, shape)
    tg, tb, td, tx = up(mt, gamma), up(mt, beta), up(mt, delta), up(mt, x)
    mt.Fused.LayerNormForward(out, tx, tg, tb, mean, ivar, pk)
    for source in (tx, pk):
        mt.Fused.LayerNormBackward(error, dg, db, td, tg, source, mean, ivar, accumulate=False)
        assert all(intact(t) for t in (out, mean, ivar, error, dg, db))
    raw = memory.numpy().ravel()
    assert (raw[:32] == 5).all() and (raw[32 + size // 4:] == 5).all()


def test_more_than_2_31_elements(mt):
    """Rows beyond element 2^31 have the bits they have in a small tensor."""
    n, rows = 1024, (1 << 21) + 5
    tail = 9
    x, gamma, beta, delta = inputs(8, (tail, 1, n, 1), (1, 1, n, 1))
    big, out, dl = (mt.CTensor(rows, 1, n, 1) for _ in range(3))
    pk = mt.CPackedTensor(rows, 1, n, 1)
    mean, ivar = mt.CTensor(rows, 1, 1, 1), mt.CTensor(rows, 1, 1, 1)
    view = lambda t: mt.CTensor.wrap(t.ptr.value + (rows - tail) * n * 4, (tail, 1, n, 1))
    mt.CTensorMath.Fill(big, 0.5)
    mt.CTensorMath.Fill(dl, 0.0)
    view(big).upload(x)
    view(dl).upload(delta)
    tg, tb = up(mt, gamma), up(mt, beta)
    mt.Fused.LayerNormForward(out, big, tg, tb, mean, ivar, pk)
    want = run_forward(mt, x, gamma, beta)
    assert np.array_equal(view(out).numpy(), want[0])
    dg, db = mt.CTensor(1, 1, n, 1), mt.CTensor(1, 1, n, 1)
    kept = po.through_8_bits(x)
    for source, v in ((big, x), (pk, kept)):
        mt.Fused.LayerNormBackward(out, dg, db, dl, tg, source, mean, ivar, accumulate=False)
        small = run_backward(mt, delta, v, gamma, beta, want[1], want[2])
        assert np.array_equal(view(out).numpy(), small["error"])
        back = po.backward(delta, v, gamma, beta, want[1], want[2], None)   # all other rows have delta 0: the sums are the tail's
        within(dg.numpy(), back, "dgamma")
        within(db.numpy(), back, "dbeta")
    mt.CTensorMath.Unpack(out, pk)
    assert np.array_equal(view(out).numpy(), kept)
    for t in (big, out, dl, pk, mean, ivar):
        t.free()


@pytest.mark.parametrize("n", [1, 2])
def test_more_rows_than_one_launch_takes(mt, n):
    """Rows of one and two values, more than 2^26 of them: 32 rows per block, at most 2^21 blocks per launch."""
    rows, tail = (1 << 26) + 77, 40
    x, gamma, beta, delta = inputs(4, (tail, 1, n, 1), (1, 1, n, 1))
    big, out = mt.CTensor(rows, 1, n, 1), mt.CTensor(rows, 1, n, 1)
    mean, ivar = mt.CTensor(rows, 1, 1, 1), mt.CTensor(rows, 1, 1, 1)
    mt.CTensorMath.Fill(big, 0.25)
    mt.CTensorMath.Fill(out, 9.0)
    view = lambda t, k=n: mt.CTensor.wrap(t.ptr.value + (rows - tail) * k * 4, (tail, 1, k, 1))
    view(big).upload(x)
    tg, tb = up(mt, gamma), up(mt, beta)
    mt.Fused.LayerNormForward(out, big, tg, tb, mean, ivar)
    want = run_forward(mt, x, gamma, beta)
    assert np.array_equal(view(out).numpy(), want[0]) and np.array_equal(view(mean, 1).numpy(), want[1]) and np.array_equal(view(ivar, 1).numpy(), want[2])
    middle = mt.CTensor.wrap(out.ptr.value + ((1 << 26) - 8) * n * 4, (16, 1, n, 1)).numpy()      # on both sides of the first launch's end
    assert np.array_equal(middle, np.broadcast_to(beta, middle.shape))                        # a constant row: xhat is 0
    view(out).upload(delta)
    mt.Fused.LayerNormBackward(out, None, None, out, tg, big, mean, ivar)
    small = run_backward(mt, delta, x, gamma, beta, want[1], want[2])
    assert np.array_equal(view(out).numpy(), small["error"])
    for t in (big, out, mean, ivar):
        t.free()
