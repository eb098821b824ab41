"""What the layer-norm and 8-bit entry points refuse: host-side checks, no device needed.  The pointers are numbers that nothing
dereferences: every call here returns before it would touch the device."""
import ctypes as C
import os

import numpy as np
import pytest

import packed_oracle as po


@pytest.fixture(scope="module")
def mt():
    import mi355tensor
    if not os.path.exists(mi355tensor.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    mi355tensor.lib()
    return mi355tensor


class Fake:
    """Descriptors over addresses far apart; nothing is there."""

    def __init__(self, mt):
        self.mt, self.at = mt, 0x10_0000_0000

    def tensor(self, *shape):
        t = self.mt.CTensor.wrap(self.at, shape)
        self.at += 0x1_0000_0000
        return t

    def packed(self, *shape):
        t = self.mt.CPackedTensor.wrap(self.at, shape)
        self.at += 0x1_0000_0000
        return t


@pytest.fixture
def fake(mt):
    return Fake(mt)


def refused(mt, code, text, f, *args, **kw):
    with pytest.raises(mt.TensorError) as e:
        f(*args, **kw)
    assert e.value.code == code and text in str(e.value), str(e.value)


SHAPE, ARGUMENT, UNAVAILABLE = 5, 6, 7


class Null:
    """A descriptor with sizes and no memory (the binding's own tensors refuse to be one); it passes for either kind."""

    def __init__(self, mt, shape):
        self.desc = mt.MtTensor(None, *shape)

    def ref(self):
        return C.byref(self.desc)


def at(mt, t, offset, shape=None):
    return mt.CTensor.wrap(t.ptr.value + offset, shape or t.shape)


def forward_args(fake):
    return [fake.tensor(4, 3, 5, 6), fake.tensor(4, 3, 5, 6), fake.tensor(1, 1, 5, 6), fake.tensor(1, 1, 5, 6), fake.tensor(4, 3, 1, 1), fake.tensor(4, 3, 1, 1), fake.packed(4, 3, 5, 6)]


def test_forward(mt, fake):
    f = mt.Fused.LayerNormForward
    good = forward_args(fake)
    out, x = good[0], good[1]
    swap = lambda i, t: good[:i] + [t] + good[i + 1:]
    for i in range(4):
        refused(mt, ARGUMENT, "null tensor", f, *swap(i, Null(mt, good[i].shape)))
    for i in (4, 5):
        refused(mt, ARGUMENT, "null tensor", f, *swap(i, Null(mt, good[i].shape)))
        for shape in ((4, 1, 1, 1), (4, 3, 5, 1), (3, 3, 1, 1), (12, 1, 1, 1)):
            refused(mt, SHAPE, "one value per row", f, *swap(i, fake.tensor(*shape)))
    for shape in ((2, 1, 5, 6), (1, 1, 5, 1), (1, 3, 1, 6), (1, 2, 5, 6), (1, 1, 4, 6), (1, 1, 1, 5), (0, 1, 5, 6)):
        refused(mt, SHAPE, "gamma", f, *swap(2, fake.tensor(*shape)))
    refused(mt, SHAPE, "sizes do not match", f, *swap(0, fake.tensor(4, 3, 6, 5)))
    refused(mt, SHAPE, "sizes do not match", f, *swap(3, fake.tensor(1, 3, 5, 6)))
    refused(mt, SHAPE, "packed", f, *swap(6, fake.packed(4, 3, 6, 5)))
    refused(mt, ARGUMENT, "16-byte", f, *swap(6, Null(mt, x.shape)))
    refused(mt, ARGUMENT, "16-byte", f, *swap(6, mt.CPackedTensor.wrap(0x5008, x.shape)))
    for func in (6, 7, 8, 9, 16, -2):
        mt.FUNC["?"] = func
        try:
            refused(mt, ARGUMENT, "function id", f, *good, func="?")
        finally:
            del mt.FUNC["?"]
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, x, 16)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, x, -4)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, good[2], 0, x.shape)))
    refused(mt, ARGUMENT, "memory", f, *swap(4, at(mt, x, 64, good[4].shape)))
    refused(mt, ARGUMENT, "memory", f, *swap(5, good[4]))
    refused(mt, ARGUMENT, "memory", f, *swap(5, at(mt, out, 0, good[5].shape)))
    for i in range(6):
        refused(mt, ARGUMENT, "memory", f, *swap(6, mt.CPackedTensor.wrap(good[i].ptr.value, x.shape)))
    refused(mt, UNAVAILABLE, "2^31", f, fake.tensor(1, 1, 1 << 16, 1 << 15), fake.tensor(1, 1, 1 << 16, 1 << 15), fake.tensor(1, 1, 1 << 16, 1 << 15), fake.tensor(1, 1, 1 << 16, 1 << 15))


@pytest.mark.parametrize("packed", [False, True])
def test_backward(mt, fake, packed):
    f = mt.Fused.LayerNormBackward
    x = (4, 3, 5, 6)
    good = [fake.tensor(*x), fake.tensor(1, 1, 1, 6), fake.tensor(1, 1, 1, 6), fake.tensor(*x), fake.tensor(1, 1, 1, 6), fake.packed(*x) if packed else fake.tensor(*x),
            fake.tensor(4, 3, 5, 1), fake.tensor(4, 3, 5, 1)]
    beta = fake.tensor(1, 1, 1, 6)
    swap = lambda i, t: good[:i] + [t] + good[i + 1:]
    wrap = mt.CPackedTensor.wrap if packed else mt.CTensor.wrap
    for i in (0, 3, 4, 6, 7):
        refused(mt, ARGUMENT, "null tensor", f, *swap(i, Null(mt, good[i].shape)))
    name = "mt_layernorm_backward_packed_func" if packed else "mt_layernorm_backward_func"
    with pytest.raises(mt.TensorError) as e:
        mt.call(name, *(t.ref() for t in good[:5]), None, Null(mt, x).ref(), good[6].ref(), good[7].ref(), C.c_int(-1), C.c_int(0))
    assert e.value.code == ARGUMENT and "null" in str(e.value)
    for i in (1, 2):
        refused(mt, SHAPE, "gradients", f, *swap(i, Null(mt, good[i].shape)))
        refused(mt, SHAPE, "gradients", f, *swap(i, fake.tensor(1, 1, 5, 6)))
    refused(mt, SHAPE, "sizes do not match", f, *swap(0, fake.tensor(4, 5, 3, 6)))
    refused(mt, SHAPE, "sizes do not match", f, *swap(5, wrap(0x9000, (4, 5, 3, 6))))
    refused(mt, SHAPE, "gamma", f, *swap(4, fake.tensor(1, 3, 5, 1)))
    for i in (6, 7):
        refused(mt, SHAPE, "one value per row", f, *swap(i, fake.tensor(4, 3, 1, 1)))
    refused(mt, SHAPE, "beta", f, *good, func="relu")
    refused(mt, SHAPE, "beta", f, *good, func="relu", beta=fake.tensor(1, 1, 5, 6))
    for func in (6, 8, 12, -5):
        mt.FUNC["?"] = func
        try:
            refused(mt, ARGUMENT, "function id", f, *good, func="?", beta=beta)
        finally:
            del mt.FUNC["?"]
    delta = good[3]
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, delta, 4)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, good[5], 0, x)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, good[4], 0, x)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, good[6], 0, x)))
    refused(mt, ARGUMENT, "memory", f, *swap(0, at(mt, beta, 0, x)), func="tangence", beta=beta)
    for i in (1, 2):
        for other in (0, 3, 4, 5, 6, 7):
            refused(mt, ARGUMENT, "memory", f, *swap(i, at(mt, good[other], 0, good[i].shape)))
    refused(mt, ARGUMENT, "memory", f, *swap(2, good[1]))


def test_packed_bytes(mt):
    b = mt.CPackedTensor.bytes_of
    assert b((1, 1, 1, 1)) == 24 and b((1, 1, 128, 1)) == 136 and b((3, 1, 129, 1)) == 3 * (144 + 16) and b((2, 3, 192, 256)) == 2 * (147456 + 8 * 1152)
    assert b((0, 1, 5, 1)) == 0 and b((4, 0, 5, 1)) == 0 and b((7, 1, 1, 0)) == 0
    assert b((1 << 31, 1, 100, 1)) == (1 << 31) * (112 + 8)
    for shape in ((1, 1, 1 << 31, 1), (1, 1 << 16, 1 << 16, 1), (1, 1 << 31, 1 << 31, 4), (1, 0xffffffff, 0xffffffff, 0xffffffff)):
        refused(mt, UNAVAILABLE, "2^31", b, shape)
    with pytest.raises(mt.TensorError) as e:
        mt.call("mt_packed_bytes", C.c_uint32(1), C.c_uint32(1), C.c_uint32(1), C.c_uint32(1), None)
    assert e.value.code == ARGUMENT


def test_pack_and_unpack(mt, fake):
    x, p = fake.tensor(2, 3, 4, 5), fake.packed(2, 3, 4, 5)
    for f, tensor_first in ((mt.CTensorMath.Pack, False), (mt.CTensorMath.Unpack, True)):
        go = lambda t, k: f(t, k) if tensor_first else f(k, t)
        refused(mt, ARGUMENT, "null", go, Null(mt, x.shape), p)
        refused(mt, ARGUMENT, "null", go, x, Null(mt, x.shape))
        refused(mt, ARGUMENT, "16-byte", go, x, mt.CPackedTensor.wrap(p.ptr.value + 8, x.shape))
        refused(mt, SHAPE, "sizes", go, x, fake.packed(2, 3, 5, 4))
        refused(mt, SHAPE, "sizes", go, x, fake.packed(3, 3, 4, 5))
        refused(mt, ARGUMENT, "memory", go, x, mt.CPackedTensor.wrap(x.ptr.value, x.shape))
        refused(mt, ARGUMENT, "memory", go, at(mt, p, p.nbytes - 4, x.shape), p)


def test_linear(mt, fake):
    f = mt.Fused.LinearBackwardWeightsSum
    good = [fake.tensor(1, 1, 7, 60), fake.tensor(1, 1, 7, 1), fake.packed(4, 3, 4, 5), fake.tensor(4, 1, 7, 1)]
    swap = lambda i, t: good[:i] + [t] + good[i + 1:]
    for i in (0, 1, 3):
        refused(mt, ARGUMENT, "null", f, *swap(i, Null(mt, good[i].shape)))
    refused(mt, ARGUMENT, "null", f, *swap(2, Null(mt, (4, 3, 4, 5))))
    for shape in ((2, 1, 7, 60), (1, 1, 60, 7), (1, 7, 1, 60), (1, 1, 7, 61), (1, 1, 8, 60)):
        refused(mt, SHAPE, "dweight", f, *swap(0, fake.tensor(*shape)))
    for shape in ((5, 1, 7, 1), (4, 1, 8, 1), (4, 7, 7, 1)):
        refused(mt, SHAPE, "delta", f, *swap(3, fake.tensor(*shape)))
    for shape in ((1, 1, 8, 1), (1, 7, 1, 1), (1, 1, 1, 7), (4, 1, 7, 1)):
        refused(mt, SHAPE, "dbias", f, *swap(1, fake.tensor(*shape)))
    for i in (0, 1):
        refused(mt, ARGUMENT, "memory", f, *swap(i, at(mt, good[2], 0, good[i].shape)))
        refused(mt, ARGUMENT, "memory", f, *swap(i, at(mt, good[3], 0, good[i].shape)))
    refused(mt, ARGUMENT, "memory", f, *swap(1, at(mt, good[0], 4 * 7 * 59, good[1].shape)))


def test_the_oracle_of_the_8_bit_form():
    """The numpy restatement against the definition: within half a step, ends exact, equal values exact."""
    x = (np.random.default_rng(1).standard_normal((5, 1, 1000, 1)) * 3 + 1).astype(np.float32)
    q, low, step = po.pack(x)
    assert q.min() == 0 and q.max() == 255
    v = po.through_8_bits(x)
    per = np.repeat(np.arange(low.shape[1]), po.GROUP)[:1000]
    assert (np.abs(v - x).reshape(5, -1) <= step[:, per] * 0.5001 + 1e-6).all()
    assert (np.abs(np.diff(v.reshape(5, -1)[:, :128])) <= 256 * step[:, :1]).all()
    c = np.full((2, 1, 200, 1), 0.1, np.float32)
    assert np.array_equal(po.through_8_bits(c), c)
    c[1, 0, 150, 0] = np.nan
    lost = np.isnan(po.through_8_bits(c))[1, 0, :, 0]
    assert not lost[:128].any() and lost[128:].all()


def test_the_oracle_of_the_norm_against_autograd():
    import torch
    x, gamma, beta, delta = (torch.from_numpy(np.random.default_rng(k).standard_normal(s)) for k, s in enumerate(((6, 3, 4, 5), (1, 1, 4, 5), (1, 1, 4, 5), (6, 3, 4, 5))))
    for t in (x, gamma, beta):
        t.requires_grad_(True)
    mean = x.mean((2, 3), keepdim=True)
    ivar = 1 / torch.sqrt(((x - mean) ** 2).mean((2, 3), keepdim=True) + float(np.float32(1e-6)))
    torch.tanh(gamma * ((x - mean) * ivar) + beta).backward(delta)
    a = [t.detach().numpy() for t in (delta, x, gamma, beta, mean, ivar)]
    got = po.backward(*a, "tangence")
    for key, t in (("error", x), ("dgamma", gamma), ("dbeta", beta)):
        assert np.allclose(got[key], t.grad.numpy(), rtol=1e-10, atol=1e-12), key
    assert np.allclose(po.forward(a[1], a[2], a[3], 1e-6, "tangence")["out"], np.tanh(a[2] * ((a[1] - a[4]) * a[5]) + a[3]), rtol=1e-12)
