"""Activations in 8 bits and the linear layer's gradient from them, on the GPU: the 8-bit form bit for bit against its
restatement in numpy, the gradient against float64."""
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


def up(mt, a):
    return mt.CTensor.from_numpy(np.ascontiguousarray(a, np.float32))


def raw(mt, pk):
    """The packed tensor's memory as the header lays it out: (bytes [W,pitch], low and step [W,groups])."""
    w, n = pk.shape[0], int(np.prod(pk.shape[1:]))
    pitch, groups = -(-n // 16) * 16, -(-n // po.GROUP)
    assert pk.nbytes == w * (pitch + 8 * groups)
    a = mt.CTensor.wrap(pk.ptr.value, (1, 1, 1, pk.nbytes // 4)).numpy().ravel()
    pairs = a[w * pitch // 4:].reshape(w, groups, 2)
    return a[:w * pitch // 4].view(np.uint8).reshape(w, pitch), pairs[:, :, 0], pairs[:, :, 1]


SHAPES = [(1, 1, 1, 1), (1, 1, 2, 1), (3, 1, 5, 1), (2, 1, 15, 1), (2, 1, 16, 1), (2, 1, 17, 1), (4, 1, 127, 1), (4, 1, 128, 1), (4, 1, 129, 1), (4, 1, 130, 1), (3, 1, 132, 1),
          (5, 1, 255, 1), (5, 1, 256, 1), (5, 3, 7, 11), (33, 1, 1001, 1), (7, 3, 32, 32), (2, 3, 192, 256), (1, 1, 100003, 1), (4000, 1, 3, 1), (70000, 1, 2, 1), (1000, 1, 260, 1),
          (1, 1, 1, 5000), (64, 64, 16, 16)]


@pytest.mark.parametrize("shape", SHAPES)
def test_pack_and_unpack(mt, shape):
    x = (Nrm(sum(shape), *shape) * 2 + 0.5).astype(np.float32)
    pk, back = mt.CPackedTensor(*shape), mt.CTensor(*shape)
    mt.CTensorMath.Pack(pk, up(mt, x))
    mt.CTensorMath.Unpack(back, pk)
    q, low, step = po.pack(x)
    gq, glow, gstep = raw(mt, pk)
    n = q.shape[1]
    assert np.array_equal(glow, low) and np.array_equal(gstep, step) and np.array_equal(gq[:, :n], q) and not gq[:, n:].any()
    values = po.unpack(q, low, step, shape)
    assert np.array_equal(back.numpy(), values)
    # |value - x| <= step/2, the rounding of (x - low) / step and of low + step*q
    per = np.repeat(np.arange(low.shape[1]), po.GROUP)[:n]
    bound = step[:, per] * (0.5 + 255 * 4 * po.U) + 3 * po.U * (np.abs(low[:, per]) + 255 * step[:, per])
    assert (np.abs(values.astype(np.float64) - x).reshape(shape[0], n) <= bound).all()


@pytest.mark.parametrize("shape", [(3, 1, 128, 1), (5, 1, 1000, 1), (7, 3, 32, 32), (3, 1, 132, 1)])
def test_past_the_caches(mt, shape):
    """What tensors of 128 MiB and more get, on small ones: the same bits."""
    x = Nrm(11, *shape)
    got = []
    for option in (0, 1):
        mt.set_option("nontemporal", option)
        try:
            pk, back = mt.CPackedTensor(*shape), mt.CTensor(*shape)
            mt.CTensorMath.Pack(pk, up(mt, x))
            mt.CTensorMath.Unpack(back, pk)
            got.append([*raw(mt, pk), back.numpy()])
        finally:
            mt.set_option("nontemporal", 2)
    assert all(np.array_equal(a, b) for a, b in zip(*got)) and np.array_equal(got[0][3], po.through_8_bits(x))


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("n", [4, 128, 1000, 1001, 4096])
def test_tensors_off_a_16_byte_boundary(mt, n, shift):
    x = Nrm(n, 5, 1, n, 1)
    whole, out = up(mt, np.concatenate([np.zeros(shift, np.float32), x.ravel()]).reshape(1, 1, 1, -1)), up(mt, np.full((1, 1, 1, 5 * n + 8), 9))
    pk = mt.CPackedTensor(5, 1, n, 1)
    mt.CTensorMath.Pack(pk, mt.CTensor.wrap(whole.ptr.value + 4 * shift, x.shape))
    mt.CTensorMath.Unpack(mt.CTensor.wrap(out.ptr.value + 4 * shift, x.shape), pk)
    got = out.numpy().ravel()
    assert np.array_equal(got[shift:shift + 5 * n].reshape(x.shape), po.through_8_bits(x))
    assert (got[:shift] == 9).all() and (got[shift + 5 * n:] == 9).all()


@pytest.mark.parametrize("n", [1, 100, 128, 300, 1024])
def test_values_that_stand_at_an_edge(mt, n):
    """Equal values come back exactly; tiny ranges as the lowest value; ties go to the even count; a group that is not finite
    comes back as NaN and its neighbours do not."""
    rows = [np.full(n, -3.7, np.float32), np.zeros(n, np.float32), np.linspace(0, 255, n, dtype=np.float32), np.float32(1e-38) * Nrm(1, n), np.float32(3e38) * np.sign(Nrm(2, n)),
            np.arange(n, dtype=np.float32) % 2 * np.float32(255) + np.float32(0.5), (np.arange(n) % 511 / 2).astype(np.float32), Nrm(3, n), Nrm(4, n), Nrm(5, n), Nrm(6, n) * np.float32(1e30)]
    rows[7][n // 2], rows[8][n // 3], rows[9][0] = np.nan, np.inf, -np.inf
    x = np.stack(rows).reshape(len(rows), 1, n, 1)
    pk, back = mt.CPackedTensor(*x.shape), mt.CTensor(*x.shape)
    mt.CTensorMath.Pack(pk, up(mt, x))
    mt.CTensorMath.Unpack(back, pk)
    got, want = back.numpy(), po.through_8_bits(x)
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(got[0], x[0]) and np.array_equal(got[1], x[1])
    g = n // 2 // po.GROUP
    inside = np.zeros(n, bool)
    inside[g * po.GROUP:(g + 1) * po.GROUP] = True
    assert np.array_equal(np.isnan(got[7].ravel()), inside)


def run_linear(mt, x, delta, accumulate=False, start=None, bias=True):
    n_in, n_out = int(np.prod(x.shape[1:])), int(np.prod(delta.shape[1:]))
    pk = mt.CPackedTensor(*x.shape)
    mt.CTensorMath.Pack(pk, up(mt, x))
    dw, db = (up(mt, np.full(s, 7, np.float32) if start is None else a) for s, a in (((1, 1, n_out, n_in), start and start[0]), ((1, 1, n_out, 1), start and start[1])))
    mt.Fused.LinearBackwardWeightsSum(dw, db if bias else None, pk, up(mt, delta), accumulate=accumulate)
    return dw.numpy().reshape(n_out, n_in), db.numpy().ravel()


def check_linear(mt, b, n_in, n_out, seed):
    x, delta = (Nrm(seed, b, 1, n_in, 1) + 0.5).astype(np.float32), Nrm(seed + 1, b, 1, n_out, 1, std=0.1)
    dw, db = run_linear(mt, x, delta)
    want = po.linear_weights(delta.reshape(b, n_out), x)
    for key, got in (("dweight", dw), ("dbias", db)):
        off = np.abs(got - want[key])
        assert (off <= want[key + "_tol"]).all(), (key, float(np.max(off / (want[key + "_tol"] + 1e-44))))
    # and as a whole: the roundings of B products are independent, so their sum grows with the root of B
    size = np.linalg.norm(np.abs(delta.reshape(b, n_out)).astype(np.float64).T @ np.abs(x.reshape(b, n_in)).astype(np.float64))
    assert np.linalg.norm(dw - want["dweight"]) <= 8 * po.U * size


@pytest.mark.parametrize("b", [1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 513, 1000])
def test_linear_batches(mt, b):
    check_linear(mt, b, 257, 130, b)


@pytest.mark.parametrize("n_in", [1, 2, 15, 16, 17, 100, 127, 128, 129, 130, 255, 256, 1000, 1024])
@pytest.mark.parametrize("n_out", [1, 3, 31, 32, 33, 64, 127, 129, 256, 257, 300])
def test_linear_sizes(mt, n_in, n_out):
    check_linear(mt, 37, n_in, n_out, n_in + n_out)


@pytest.mark.parametrize("b,n_in,n_out", [(32, 1024, 6144), (256, 4096, 768), (4096, 512, 512), (3000, 1000, 100), (20000, 64, 48), (5000, 16, 1000), (640, 2048, 2048)])
def test_linear_large(mt, b, n_in, n_out):
    check_linear(mt, b, n_in, n_out, b)


def unequal(x, delta, what):
    """Magnitudes that 16 bits cannot hold beside one another."""
    rng = np.random.default_rng(5)
    if what == "samples without delta":        # as padding may leave them: huge activations, no gradient
        x[3], delta[3] = x[3] * 1e30, 0
        x[-1], delta[-1] = x[-1] * 1e12, 0
    elif what == "samples with little delta":
        x[3], delta[3] = x[3] * 1e10, delta[3] * 1e-10
    elif what == "one feature's activations":
        x[:, :, 5] *= 1e8
    elif what == "every row":
        delta *= np.exp(rng.uniform(-60, 60, (1, delta.shape[1], delta.shape[2], 1))).astype(np.float32)
    elif what == "every sample":
        x *= np.exp(rng.uniform(-25, 25, (x.shape[0], 1, 1, 1))).astype(np.float32)
    elif what == "rows of zeros":
        delta[:, :, ::3] = 0
    elif what == "one sample of a row":
        delta[:, :, 7] = 0
        delta[11, :, 7] = 1e-20
    elif what == "constant activations":
        x[:, :, :128] = x[:, :, :1]


# the first three are large enough for two fp16 numbers per product (256 rows per block, 128, an odd number of them in parts of the batch)
@pytest.mark.parametrize("b,n_in,n_out", [(1100, 4000, 4000), (1500, 2000, 1500), (5000, 1000, 1501), (300, 257, 130)])
@pytest.mark.parametrize("what", ["nothing", "samples without delta", "samples with little delta", "one feature's activations", "every row", "every sample",
                                  "rows of zeros", "one sample of a row", "constant activations"])
def test_linear_unequal_magnitudes(mt, b, n_in, n_out, what):
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1, std=0.02)
    unequal(x, delta, what)
    dw, db = run_linear(mt, x, delta)
    want = po.linear_weights(delta.reshape(b, n_out), x)
    for key, got in (("dweight", dw), ("dbias", db)):
        assert (np.abs(got - want[key]) <= want[key + "_tol"] + 1e-44).all(), (key, float(np.max(np.abs(got - want[key]) / (want[key + "_tol"] + 1e-44))))
    # and every row as a whole, as in check_linear
    size = want["dweight_tol"] / (b + 18)
    assert (np.linalg.norm(dw - want["dweight"], axis=1) <= 8 * np.linalg.norm(size, axis=1) + 1e-44).all()
    again = run_linear(mt, x, delta)
    assert np.array_equal(dw, again[0]) and np.array_equal(db, again[1])
    added = run_linear(mt, x, delta, accumulate=True, start=(np.ones((1, 1, n_out, n_in), np.float32), np.ones((1, 1, n_out, 1), np.float32)))
    assert np.array_equal(added[0], dw + np.float32(1)) and np.array_equal(added[1], db + np.float32(1))


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("b,n_in,n_out", [(40, 300, 140), (300, 260, 128), (1500, 2000, 1500)])
def test_linear_off_a_16_byte_boundary(mt, b, n_in, n_out, shift):
    """delta, dweight and dbias `shift` floats behind a 16-byte boundary: the same bits, nothing written beside them."""
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1)
    want = run_linear(mt, x, delta)
    pk = mt.CPackedTensor(*x.shape)
    mt.CTensorMath.Pack(pk, up(mt, x))
    held = []
    for a, shape in ((delta, delta.shape), (None, (1, 1, n_out, n_in)), (None, (1, 1, n_out, 1))):
        n = int(np.prod(shape))
        whole = up(mt, np.concatenate([np.full(shift, 9), np.full(n, 7) if a is None else a.ravel(), np.full(8, 9)]).reshape(1, 1, 1, -1))
        held.append((whole, mt.CTensor.wrap(whole.ptr.value + 4 * shift, shape), n))
    mt.Fused.LinearBackwardWeightsSum(held[1][1], held[2][1], pk, held[0][1], accumulate=False)
    for (whole, _, n), w in zip(held[1:], want):
        got = whole.numpy().ravel()
        assert np.array_equal(got[shift:shift + n], w.ravel()) and (got[:shift] == 9).all() and (got[shift + n:] == 9).all()


@pytest.mark.parametrize("b,n_in,n_out", [(5, 100, 30), (300, 257, 129), (4096, 128, 64), (64, 1024, 1024)])
def test_linear_adds_and_repeats(mt, b, n_in, n_out):
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, n_out, 1, 1)      # delta seen as [B,Out,1,1]
    start = (Nrm(3, 1, 1, n_out, n_in), Nrm(4, 1, 1, n_out, 1))
    fresh, again = run_linear(mt, x, delta), run_linear(mt, x, delta)
    assert all(np.array_equal(a, c) for a, c in zip(fresh, again))
    added = run_linear(mt, x, delta, accumulate=True, start=start)
    assert np.array_equal(added[0], start[0].reshape(n_out, n_in) + fresh[0]) and np.array_equal(added[1], start[1].ravel() + fresh[1])
    alone = run_linear(mt, x, delta, bias=False)
    assert np.array_equal(alone[0], fresh[0]) and (alone[1] == 7).all()


@pytest.mark.parametrize("b,n_in,n_out", [(40, 300, 140), (3000, 130, 60), (1500, 2000, 1500), (1100, 4000, 4000)])
def test_linear_values_that_are_not_finite(mt, b, n_in, n_out):
    x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1)
    fine = run_linear(mt, x, delta)
    bad = delta.copy()
    bad[b - 1, 0, 5, 0], bad[0, 0, 7, 0] = np.inf, np.nan
    dw, db = run_linear(mt, x, bad)
    others = [o for o in range(n_out) if o not in (5, 7)]
    assert not np.isfinite(dw[[5, 7]]).any() and np.isinf(db[5]) and np.isnan(db[7])
    assert np.array_equal(dw[others], fine[0][others]) and np.array_equal(db[others], fine[1][others])
    bad_x = x.copy()
    bad_x[b - 1, 0, 129, 0] = np.nan                       # a group's elements are lost together: columns 128 ... 255
    dw, db = run_linear(mt, bad_x, delta)
    lost = slice(128, min(256, n_in))
    assert np.isnan(dw[:, lost]).all() and np.array_equal(np.delete(dw, np.r_[lost], 1), np.delete(fine[0], np.r_[lost], 1)) and np.array_equal(db, fine[1])


@pytest.mark.parametrize("scale", [1e-20, 1e15])
def test_linear_scales(mt, scale):
    x, delta = Nrm(1, 70, 1, 200, 1), (Nrm(2, 70, 1, 90, 1) * scale).astype(np.float32)
    dw, _ = run_linear(mt, x, delta)
    want = po.linear_weights(delta.reshape(70, 90), x)
    assert (np.abs(dw - want["dweight"]) <= want["dweight_tol"]).all()


def test_linear_of_nothing(mt):
    start = (np.full((1, 1, 5, 6), 2, np.float32), np.full((1, 1, 5, 1), 3, np.float32))
    x, delta = np.zeros((0, 1, 6, 1), np.float32), np.zeros((0, 1, 5, 1), np.float32)
    kept = run_linear(mt, x, delta, accumulate=True, start=start)
    assert (kept[0] == 2).all() and (kept[1] == 3).all()
    none = run_linear(mt, x, delta)
    assert not none[0].any() and not none[1].any()
    db = run_linear(mt, np.zeros((4, 1, 0, 1), np.float32), np.ones((4, 1, 5, 1), np.float32))[1]     # no input features: the bias has its gradient
    assert (db == 4).all()


def test_linear_writes_its_gradients_only(mt):
    for b, n_in, n_out in ((9, 130, 70), (2000, 200, 33)):
        x, delta = Nrm(1, b, 1, n_in, 1), Nrm(2, b, 1, n_out, 1)
        memory = up(mt, np.full((1, 1, 1, n_out * n_in + n_out + 192), 5))
        dw = mt.CTensor.wrap(memory.ptr.value + 4 * 64, (1, 1, n_out, n_in))
        db = mt.CTensor.wrap(memory.ptr.value + 4 * (128 + n_out * n_in), (1, 1, n_out, 1))
        pk = mt.CPackedTensor(*x.shape)
        mt.CTensorMath.Pack(pk, up(mt, x))
        mt.Fused.LinearBackwardWeightsSum(dw, db, pk, up(mt, delta), accumulate=False)
        a = memory.numpy().ravel()
        assert (a[:64] == 5).all() and (a[64 + n_out * n_in:128 + n_out * n_in] == 5).all() and (a[128 + n_out * n_in + n_out:] == 5).all()


def make_step(mt, b, n_in, n_hidden, n_out, seed=1):
    """A block of a network as it would be trained: linear, layer norm + leaky ReLU that keeps its input in 8 bits, linear whose
    input is kept in 8 bits."""
    T = mt.CTensor
    p = {"w1": Nrm(seed, 1, 1, n_hidden, n_in, std=n_in ** -0.5), "b1": Nrm(seed + 1, 1, 1, n_hidden, 1, std=0.1), "gamma": (1 + 0.1 * Nrm(seed + 2, 1, 1, n_hidden, 1)).astype(np.float32),
         "beta": Nrm(seed + 3, 1, 1, n_hidden, 1, std=0.1), "w2": Nrm(seed + 4, 1, 1, n_out, n_hidden, std=n_hidden ** -0.5), "b2": Nrm(seed + 5, 1, 1, n_out, 1, std=0.1)}
    x, delta = Nrm(seed + 6, b, 1, n_in, 1), Nrm(seed + 7, b, 1, n_out, 1, std=0.1)
    t = {k: up(mt, v) for k, v in p.items()}
    t.update(x=up(mt, x), delta=up(mt, delta), h=T(b, 1, n_hidden, 1), a=T(b, 1, n_hidden, 1), y=T(b, 1, n_out, 1), mean=T(b, 1, 1, 1), ivar=T(b, 1, 1, 1),
             da=T(b, 1, n_hidden, 1), dh=T(b, 1, n_hidden, 1), dx=T(b, 1, n_in, 1), kx=mt.CPackedTensor(b, 1, n_in, 1), kh=mt.CPackedTensor(b, 1, n_hidden, 1), ka=mt.CPackedTensor(b, 1, n_hidden, 1))
    t.update({"d" + k: T(*v.shape) for k, v in p.items()})

    def step():
        F, M = mt.Fused, mt.CTensorMath
        M.Pack(t["kx"], t["x"])
        F.LinearForward(t["h"], t["w1"], t["x"], t["b1"])
        F.LayerNormForward(t["a"], t["h"], t["gamma"], t["beta"], t["mean"], t["ivar"], t["kh"], func="tangence")
        M.Pack(t["ka"], t["a"])
        F.LinearForward(t["y"], t["w2"], t["a"], t["b2"])
        F.LinearBackwardWeightsSum(t["dw2"], t["db2"], t["ka"], t["delta"], accumulate=False)
        M.TransponseMul(t["da"], t["w2"], t["delta"])
        F.LayerNormBackward(t["dh"], t["dgamma"], t["dbeta"], t["da"], t["gamma"], t["kh"], t["mean"], t["ivar"], beta=t["beta"], func="tangence", accumulate=False)
        F.LinearBackwardWeightsSum(t["dw1"], t["db1"], t["kx"], t["dh"], accumulate=False)
        M.TransponseMul(t["dx"], t["w1"], t["dh"])

    return p, x, delta, t, step


RESULTS = ("y", "dw2", "db2", "dgamma", "dbeta", "dw1", "db1", "dx")


@pytest.mark.parametrize("b,n_in,n_hidden,n_out", [(48, 300, 500, 70), (257, 1024, 1024, 100)])
def test_a_training_step(mt, b, n_in, n_hidden, n_out):
    """All of it together, against float64 on the values that the 8 bits stand for."""
    p, x, delta, t, step = make_step(mt, b, n_in, n_hidden, n_out)
    step()
    d = {k: v.astype(np.float64).reshape(v.shape[2], v.shape[3]) for k, v in p.items()}
    h32, a32, mean, ivar = (t[k].numpy().reshape(b, -1) for k in ("h", "a", "mean", "ivar"))
    h = x.reshape(b, -1).astype(np.float64) @ d["w1"].T + d["b1"].T
    a = np.tanh(d["gamma"].T * (h - h.mean(1, keepdims=True)) / np.sqrt(h.var(1, keepdims=True) + 1e-6) + d["beta"].T)
    dl = delta.reshape(b, -1).astype(np.float64)
    got = {k: t[k].numpy().astype(np.float64) for k in RESULTS}
    near = lambda key, want: np.linalg.norm(got[key].reshape(want.shape) - want) <= 1e-5 * np.linalg.norm(want)   # chains of four fp32 sums of up to 1024 terms
    assert near("y", a @ d["w2"].T + d["b2"].T)
    kept_a, kept_h, kept_x = (po.through_8_bits(v).astype(np.float64) for v in (a32, h32, x.reshape(b, -1)))
    assert near("dw2", dl.T @ kept_a) and near("db2", dl.sum(0))
    xhat = (kept_h - mean) * ivar
    g = (dl @ d["w2"]) * (1 - np.tanh(d["gamma"].T * xhat + d["beta"].T) ** 2)
    assert near("dgamma", (g * xhat).sum(0)) and near("dbeta", g.sum(0))
    u = g * d["gamma"].T
    dh = ivar * (u - u.mean(1, keepdims=True) - xhat * (u * xhat).mean(1, keepdims=True))
    assert near("dw1", dh.T @ kept_x) and near("db1", dh.sum(0)) and near("dx", dh @ d["w1"])
    # and how far the 8 bits move the gradients from those of fp32 activations: a step is 1/255 of a range of about six standard
    # deviations, its rounding uniform, so an activation is off by 6/255/sqrt(12) = 0.7 % of its spread; three such factors meet
    xh = (h - h.mean(1, keepdims=True)) * ivar
    g = (dl @ d["w2"]) * (1 - np.tanh(d["gamma"].T * xh + d["beta"].T) ** 2)
    u = g * d["gamma"].T
    dh = ivar * (u - u.mean(1, keepdims=True) - xh * (u * xh).mean(1, keepdims=True))
    for key, want in (("dw2", dl.T @ a), ("dgamma", (g * xh).sum(0)), ("dw1", dh.T @ x.reshape(b, -1)), ("dx", dh @ d["w1"])):
        assert np.linalg.norm(got[key].reshape(want.shape) - want) <= 0.05 * np.linalg.norm(want), key


@pytest.mark.parametrize("b,n_in,n_hidden,n_out", [(130, 700, 1024, 90), (1500, 2000, 2001, 1500)])
def test_a_recorded_step_replays(mt, b, n_in, n_hidden, n_out):
    """Recorded once, replayed with new inputs, with eager work of other sizes on the same workspaces between the replays."""
    _, x, _, t, step = make_step(mt, b, n_in, n_hidden, n_out)
    other = make_step(mt, 77, 300, 2500, 33, seed=40)[4]
    step()
    other()
    mt.synchronize()
    graph = mt.Graph(step)
    for k in range(4):
        t["x"].upload(Nrm(500 + k, *x.shape))
        graph.launch()
        replayed = {key: t[key].numpy() for key in RESULTS}
        other()
        step()
        assert all(np.array_equal(t[key].numpy(), replayed[key]) for key in RESULTS), k


def test_another_stream(mt):
    """The work follows mt_set_stream."""
    import ctypes as C
    _, x, _, t, step = make_step(mt, 40, 200, 1000, 30)
    step()
    want = {key: t[key].numpy() for key in RESULTS}
    hip, stream = C.CDLL("libamdhip64.so"), C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), C.c_uint(1)) == 0
    mt.set_stream(stream.value)
    try:
        for key in RESULTS:
            mt.CTensorMath.Fill(t[key], 9.0)
        step()
        got = {key: t[key].numpy() for key in RESULTS}
    finally:
        mt.set_stream(None)
        hip.hipStreamDestroy(stream)
    assert all(np.array_equal(got[k], want[k]) for k in RESULTS)


@pytest.mark.parametrize("batch", [4, 16])
def test_a_discriminator_with_activations_in_8_bits(mt, batch):
    """The discriminator's training step with its activations kept in 8 bits: the gradients of the ordinary step on activations that
    went through 8 bits, bit for bit but for the linear layer's product; and near those of the fp32 step."""
    import discriminator as D
    params = D.make_parameters()
    x, labels = D.make_batch(batch)
    plain, packed = D.Discriminator(batch, params), D.PackedDiscriminator(batch, params)
    for net in (plain, packed):
        net.set_batch(x, labels)
        net.forward(True)
    assert np.array_equal(plain.prob.numpy(), packed.prob.numpy())
    plain.backward(True)
    fp32 = {k: t.numpy().astype(np.float64) for k, t in plain.g.items()}
    for t in plain.a + plain.xhat:
        kept = mt.CPackedTensor(*t.shape)
        mt.CTensorMath.Pack(kept, t)
        mt.CTensorMath.Unpack(t, kept)
    plain.backward(True)
    packed.backward()
    for k in plain.g:
        a, b = plain.g[k].numpy().astype(np.float64), packed.g[k].numpy().astype(np.float64)
        # fp32 sums of `batch` products in two orders: 2 * batch roundings of sums that are at most batch times their terms
        assert np.array_equal(a, b) if not k.startswith("lin") else np.linalg.norm(a - b) <= 2 * batch * batch * po.U * np.linalg.norm(a), k
    assert np.array_equal(plain.d_x.numpy(), packed.d_x.numpy())
    # xhat within 1/255 of a range of seven deviations turns the sign of gamma*xhat+beta, and so the slope of the leaky ReLU from 0.1 to
    # 1, for 0.4 * 2 * 7/255/4 = 0.5 % of the values of a layer: 0.9 / 0.7 * sqrt(0.005) = 9 % of a delta's norm per layer, 18 % over four
    for k, want in fp32.items():
        got = packed.g[k].numpy().astype(np.float64)
        if not k.startswith("bias"):                # in front of a batch norm a bias has no gradient but rounding
            assert np.linalg.norm(got - want) <= 0.25 * np.linalg.norm(want), k
    # all but the images: 1 + 8/128 bytes per value instead of 4 (every sample is a whole number of groups)
    images = 4 * plain.x.count
    assert 64 * (packed.kept_bytes() - images) == 17 * (plain.kept_bytes() - images)
    packed.update(fused=True)
    packed.step()
    assert all(np.isfinite(t.numpy()).all() for t in packed.p.values())
