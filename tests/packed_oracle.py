"""Layer normalisation and the 8-bit form of activations restated in numpy: the 8-bit form in fp32, operation by operation
(results are compared bit for bit), the rest in float64 together with a bound of what fp32 arithmetic may add."""
import numpy as np

U = 2.0 ** -24        # half a step of fp32, relative to the value
GROUP = 128
F32 = np.float32


def pack(x):
    """(q [W,n] uint8, low [W,groups], step [W,groups]) of an fp32 tensor."""
    x = np.asarray(x, F32)
    w = x.shape[0]
    flat = x.reshape(w, -1)
    n = flat.shape[1]
    groups = -(-n // GROUP)
    q = np.zeros((w, n), np.uint8)
    low, step = np.zeros((w, groups), F32), np.zeros((w, groups), F32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = flat[:, g * GROUP:(g + 1) * GROUP]
            lo, hi = part.min(1), part.max(1)                     # numpy lets a NaN through
            span = hi - lo
            finite = span <= np.finfo(F32).max
            st = np.where(finite, span * (F32(1) / F32(255)), F32(0)).astype(F32)
            st[st < np.finfo(F32).tiny] = 0
            inverse = np.where(st > 0, F32(1) / np.where(st > 0, st, F32(1)), F32(0)).astype(F32)
            t = np.rint((part - lo[:, None]) * inverse[:, None])
            t[~np.isfinite(t)] = 0                                # the group is NaN whatever q is
            q[:, g * GROUP:(g + 1) * GROUP] = np.minimum(t, 255).astype(np.uint8)
            low[:, g], step[:, g] = np.where(finite, lo, F32(np.nan)), st
    return q, low, step


def unpack(q, low, step, shape):
    per = np.repeat(np.arange(low.shape[1]), GROUP)[:q.shape[1]]
    return (low[:, per] + step[:, per] * q.astype(F32)).astype(F32).reshape(shape)


def through_8_bits(x):
    return unpack(*pack(x), np.shape(x))


def row_view(shape, parameter_shape):
    """(rows, N, shape of a statistic) of a norm whose parameters have `parameter_shape`."""
    n = int(np.prod(parameter_shape))
    span = [p == s for p, s in zip(parameter_shape[1:], shape[1:])]
    axes = 3 if all(span) else 2 if parameter_shape[1] == 1 and span[1] and span[2] else 1
    return int(np.prod(shape)) // max(n, 1), n, tuple(shape[:4 - axes]) + (1,) * axes


def func(name, v):
    if name is None or name == "linear":
        return v
    if name == "relu":
        return np.maximum(v, 0)
    if name == "leaky_relu":
        return np.where(v > 0, v, 0.1 * v)
    c = np.clip(v, -30, 30)
    if name == "sigmoid":
        return 1 / (1 + np.exp(-c))
    if name == "tangence":
        return np.tanh(c)
    assert name == "gelu"
    return 0.5 * v * (1 + np.tanh(np.sqrt(2 / 3.141592654) * (v + 0.044715 * v ** 3)))


def derivative(name, v):
    """The framework's own derivative functions; for gelu its formula (cpu/ctensorapplyfunc.h:158-170)."""
    if name is None or name == "linear":
        return np.ones_like(v)
    if name in ("relu", "leaky_relu"):
        return np.where(v >= 0, 1.0, 0.0 if name == "relu" else 0.1)
    f = func(name, v)
    if name == "sigmoid":
        return f * (1 - f)
    if name == "tangence":
        return 1 - f * f
    a = np.sqrt(2 / 3.141592654)
    inner = a * (v + 0.044715 * v ** 3)
    return 0.5 * ((1 + np.tanh(inner)) + 0.5 * v / np.cosh(inner) ** 2) * a * (1 + 3 * 0.044715 * v * v)


# Sigmoid and tangence take the hardware's exponential and reciprocal: 3e-7 absolute (the header's figure); their
# derivatives f(1-f) and 1-f^2 at most twice that.  The largest slopes: of gelu and its derivative formula below 1.2 and 2.
def _slack(name):
    return 3e-7 if name in ("sigmoid", "tangence") else 1e-6 if name == "gelu" else 0.0


def _additions(n):
    """Additions that one value passes through in a sum of n: at most n/256 in one thread and 40 between threads and blocks."""
    return n / 256 + 40


def forward(x, gamma, beta, eps, name):
    """{out, mean, ivar} in float64 and the bounds {.._tol}."""
    rows, n, stat = row_view(x.shape, gamma.shape)
    f, g, b = x.astype(np.float64).reshape(rows, n), gamma.astype(np.float64).reshape(1, n), beta.astype(np.float64).reshape(1, n)
    d = _additions(n)
    mean = f.mean(1, keepdims=True)
    dev = f - mean
    var = (dev ** 2).mean(1, keepdims=True)
    ivar = 1 / np.sqrt(var + float(F32(eps)))
    xhat = dev * ivar
    pre = g * xhat + b
    e_mean = (d + 1) * U * np.abs(f).mean(1, keepdims=True)
    # every deviation carries e_mean and its own rounding; the sum of the deviations is zero, so e_mean enters squared
    e_var = (d + 4) * U * var + e_mean ** 2 + 2 * U * np.abs(dev).mean(1, keepdims=True) * e_mean
    e_ivar = ivar * (0.5 * e_var * ivar ** 2 + 3 * U)
    e_xhat = ivar * (e_mean + U * np.abs(dev)) + np.abs(dev) * e_ivar + U * np.abs(xhat)
    e_pre = np.abs(g) * e_xhat + U * np.abs(g * xhat) + U * np.abs(pre)
    out = func(name, pre)
    e_out = (1.2 if name == "gelu" else 1.0) * e_pre + 2 * U * np.abs(out) + _slack(name)
    shape = x.shape
    return {"out": out.reshape(shape), "mean": mean.reshape(stat), "ivar": ivar.reshape(stat),
            "out_tol": e_out.reshape(shape), "mean_tol": e_mean.reshape(stat), "ivar_tol": e_ivar.reshape(stat)}


def backward(delta, x, gamma, beta, mean, ivar, name):
    """{error, dgamma, dbeta} in float64 from the fp32 x (or the unpacked values), mean and ivar, and the bounds."""
    rows, n, _ = row_view(x.shape, gamma.shape)
    v = lambda a, *s: a.astype(np.float64).reshape(*s)
    f, dl, g, b, m, iv = v(x, rows, n), v(delta, rows, n), v(gamma, 1, n), v(beta, 1, n), v(mean, rows, 1), v(ivar, rows, 1)
    xhat = (f - m) * iv
    pre = g * xhat + b
    slope = derivative(name, pre)
    front = dl * slope
    u = front * g
    c1, c2 = u.mean(1, keepdims=True), (u * xhat).mean(1, keepdims=True)
    error = iv * (u - c1 - xhat * c2)
    d, dr = _additions(n), rows / 4 + 16
    e_xhat = 2 * U * np.abs(xhat)
    e_pre = np.abs(g) * e_xhat + U * np.abs(g * xhat) + U * np.abs(pre)
    e_slope = {None: 0.0, "linear": 0.0, "relu": 1.0, "leaky_relu": 0.9}.get(name)
    if e_slope is None:
        e_slope = 2 * e_pre + 2 * _slack(name) + 2 * U
    else:
        e_slope = np.where(np.abs(pre) <= e_pre, e_slope, 0.0) + (U if name == "leaky_relu" else 0.0)   # on which side of zero
    e_front = np.abs(dl) * e_slope + U * np.abs(front)
    e_u = np.abs(g) * e_front + U * np.abs(u)
    e_c1 = e_u.mean(1, keepdims=True) + (d + 1) * U * np.abs(u).mean(1, keepdims=True)
    e_c2 = (e_u * np.abs(xhat) + np.abs(u) * e_xhat).mean(1, keepdims=True) + (d + 2) * U * np.abs(u * xhat).mean(1, keepdims=True)
    e_error = iv * (e_u + e_c1 + np.abs(xhat) * e_c2 + e_xhat * np.abs(c2) + 4 * U * (np.abs(u) + np.abs(c1) + np.abs(xhat * c2)))
    e_dg = (e_front * np.abs(xhat) + np.abs(front) * e_xhat + (dr + 2) * U * np.abs(front * xhat)).sum(0)
    e_db = (e_front + (dr + 1) * U * np.abs(front)).sum(0)
    ps = gamma.shape
    return {"error": error.reshape(x.shape), "dgamma": (front * xhat).sum(0).reshape(ps), "dbeta": front.sum(0).reshape(ps),
            "error_tol": e_error.reshape(x.shape), "dgamma_tol": e_dg.reshape(ps), "dbeta_tol": e_db.reshape(ps)}


def linear_weights(delta, x):
    """dweight [Out,In], dbias [Out] in float64 from delta [B,Out] and the 8-bit form of x [B,In], and the bounds: one rounding
    of delta * step, and at most B + 16 additions of the products on the way to a sum."""
    q, low, step = pack(x)
    b, n = q.shape
    per = np.repeat(np.arange(low.shape[1]), GROUP)[:n]
    lo, st = low[:, per].astype(np.float64), step[:, per].astype(np.float64)
    d = delta.astype(np.float64)
    size = np.abs(lo) + st * q
    return {"dweight": d.T @ (lo + st * q), "dbias": d.sum(0), "dweight_tol": (b + 18) * U * (np.abs(d).T @ size), "dbias_tol": (b + 16) * U * np.abs(d).sum(0)}
