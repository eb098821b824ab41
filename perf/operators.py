"""Layer normalisation and activations kept in 8 bits: the cases they are measured on and their plain forms.

A case is one pass of a training or serving program through one operator:

    norm    forward pass of a layer norm (output, mean and 1/sqrt(variance + epsilon) of every row)
    back    its backward pass from the input and the statistics that the forward pass left
    step    forward pass that leaves the input in 8 bits, then the backward pass from those 8 bits
    pack    an activation put into 8 bits and, for the backward pass, back into fp32
    linear  a linear layer's input put into 8 bits, then the weight and bias gradient from them

Sizes are [w,z,y,x] as everywhere in the framework; `axes` says how many of the last sizes one row of the norm spans.
"""
import os
import sys

import torch

own = False

EPSILON = 1e-6
GROUP = 128            # consecutive elements of a sample that share a lowest value and a step
MOST = 25_000_000      # elements of the largest activation that is drawn
MOST_PRODUCTS = 1.4e11


def _norm(name, kind, w, z, y, x, axes, func="none"):
    return {"name": name, "kind": kind, "w": w, "z": z, "y": y, "x": x, "axes": axes, "func": func}


def listed():
    return [
        # one vector of 1024 features: a generator or decoder run for a single sample, where latency is everything
        _norm("norm_one", "norm", 1, 1, 1024, 1, 2),
        # a large batch of feature vectors
        _norm("norm_rows", "norm", 8192, 1, 4096, 1, 2),
        # whole images as rows: the 192x256 colour images of the GAN models, batch 32
        _norm("norm_image", "norm", 32, 3, 192, 256, 3, "sigmoid"),
        # a small batch of an odd number of features
        _norm("back_small", "back", 33, 1, 1001, 1, 2),
        # a large batch, the two gradients summed over 8192 rows
        _norm("back_rows", "back", 8192, 1, 2048, 1, 2),
        # feature maps of 16 channels as rows, with the function behind the norm
        _norm("back_image", "back", 32, 16, 96, 128, 3, "tangence"),
        # an odd number of rows along X alone, whose groups of 128 elements do not end with the rows
        _norm("step_odd", "step", 205, 1, 5, 1000, 1),
        # a training step's norm at the widest linear layer of the GAN generator
        _norm("step_rows", "step", 4096, 1, 6144, 1, 2),
        # hidden activations of an odd width
        {"name": "pack_small", "kind": "pack", "w": 65, "z": 1, "y": 1001, "x": 1},
        # feature maps of a convolution stack at batch 256
        {"name": "pack_maps", "kind": "pack", "w": 256, "z": 64, "y": 32, "x": 32},
        # the GAN generator's linear layer at its batch of 32: few samples, many weights
        {"name": "linear_gan", "kind": "linear", "w": 32, "in": 1024, "out": 6144},
        # a linear layer over many rows, where the product is the work
        {"name": "linear_rows", "kind": "linear", "w": 4096, "in": 4096, "out": 4096},
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of its range."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "back", "step", "pack", "linear"])
    if kind == "linear":
        w, n_in, n_out = _spread(rng, 1, 8192), _spread(rng, 16, 6144), _spread(rng, 8, 6144)
        if 2.0 * w * n_in * n_out > MOST_PRODUCTS:
            w = max(1, int(MOST_PRODUCTS / (2.0 * n_in * n_out)))
        return {"kind": kind, "w": w, "in": n_in, "out": n_out}
    n = _spread(rng, 16, 200000)
    rows = _spread(rng, 1, max(1, min(60000, MOST // n)))
    axes = rng.choice([1, 2, 3])
    if axes == 1:                                    # rows over W, Z and Y
        z = rng.choice([1, 1, 2, 3])
        y = rng.choice([1, 2, 5])
        w, x = max(1, rows // (z * y)), n
    elif axes == 2:                                  # feature vectors, or planes
        z = rng.choice([1, 1, 3])
        x = rng.choice([1, 1, 2, 7, 16])
        w, y = max(1, rows // z), max(1, n // x)
    else:
        z = rng.choice([1, 3, 16])
        x = rng.choice([1, 4, 9, 32])
        w, y = rows, max(1, n // (z * x))
    case = {"kind": kind, "w": w, "z": z, "y": y, "x": x}
    if kind != "pack":
        case["axes"] = axes
        case["func"] = rng.choice(["none", "none", "sigmoid", "tangence"])
    return case


def _sizes(case):
    """(rows, N) of a norm."""
    dims = (case["z"], case["y"], case["x"])
    n = 1
    for d in dims[3 - case["axes"]:]:
        n *= d
    return case["w"] * case["z"] * case["y"] * case["x"] // n, n


def _parameter_shape(case):
    dims = (case["z"], case["y"], case["x"])
    return (1,) + (1,) * (3 - case["axes"]) + dims[3 - case["axes"]:]


def _row_shape(case):
    dims = (case["z"], case["y"], case["x"])
    return (case["w"],) + dims[:3 - case["axes"]] + (1,) * case["axes"]


def _bindings():
    if "mi355tensor" not in sys.modules:
        sys.path.insert(0, os.path.abspath("cuda-cnn-gan-vae_amd"))
    import mi355tensor
    return mi355tensor


def _random(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def prepare(case, seed):
    """Inputs, and the tensors that a layer keeps for its results.  Activations have the offsets and the unequal spreads of
    real features; a linear layer's input is what a leaky ReLU leaves."""
    g = _random(seed)
    s = {"case": case}
    if case["kind"] == "linear":
        b, n_in, n_out = case["w"], case["in"], case["out"]
        x = _normal(g, b, 1, n_in, 1) + 0.3 * _normal(g, 1, 1, n_in, 1)
        s["x"] = torch.where(x > 0, x, 0.1 * x)
        s["delta"] = _normal(g, b, 1, n_out, 1) * 0.02
        s["dweight"], s["dbias"] = torch.empty(1, 1, n_out, n_in, device="cuda"), torch.empty(1, 1, n_out, 1, device="cuda")
    else:
        shape = (case["w"], case["z"], case["y"], case["x"])
        s["x"] = _normal(g, *shape) * 1.5
        if case["kind"] == "pack":
            s["x"] += 0.5
            s["out"] = torch.empty(shape, device="cuda")
        else:
            p = _parameter_shape(case)
            s["x"] += _normal(g, *p) + 0.7
            s["gamma"], s["beta"] = 1.0 + 0.2 * _normal(g, *p), 0.1 * _normal(g, *p)
            s["mean"], s["ivar"] = torch.empty(_row_shape(case), device="cuda"), torch.empty(_row_shape(case), device="cuda")
            if case["kind"] != "back":
                s["out"] = torch.empty(shape, device="cuda")
            if case["kind"] != "norm":
                s["delta"] = _normal(g, *shape) * 0.1
                s["error"] = torch.empty(shape, device="cuda")
                s["dgamma"], s["dbeta"] = torch.empty(p, device="cuda"), torch.empty(p, device="cuda")
            if case["kind"] == "back":
                mean, ivar = _statistics(case, s["x"])
                s["mean"].copy_(mean.view(_row_shape(case)))
                s["ivar"].copy_(ivar.view(_row_shape(case)))
    if own:  # the same memory under the framework's own descriptors, and the 8-bit tensor that the layer keeps
        mt = _bindings()
        mt.init(0)
        s["t"] = {k: mt.CTensor.wrap(v.data_ptr(), v.shape) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if case["kind"] in ("step", "pack", "linear"):
            s["packed"] = mt.CPackedTensor(*s["x"].shape)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _statistics(case, x):
    """Mean and 1/sqrt(variance + epsilon) of every row, [rows, 1]."""
    rows, n = _sizes(case)
    x = x.reshape(rows, n)
    mean = x.mean(1, keepdim=True)
    d = x - mean
    return mean, 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPSILON)


def _func(func, v):
    if func == "none":
        return v
    v = v.clamp(-30.0, 30.0)
    return torch.tanh(v) if func == "tangence" else 1.0 / (1.0 + torch.exp(-v))


def _derivative(func, v):
    f = _func(func, v)
    return 1.0 - f * f if func == "tangence" else (1.0 - f) * f


def _forward(case, x, gamma, beta):
    rows, n = _sizes(case)
    mean, ivar = _statistics(case, x)
    xhat = (x.view(rows, n) - mean) * ivar
    return _func(case["func"], gamma.view(1, n) * xhat + beta.view(1, n)).view_as(x), mean, ivar


def _backward(case, delta, x, gamma, beta, mean, ivar):
    rows, n = _sizes(case)
    gamma, beta, mean, ivar = gamma.view(1, n), beta.view(1, n), mean.view(rows, 1), ivar.view(rows, 1)
    xhat = (x.reshape(rows, n) - mean) * ivar
    g = delta.view(rows, n)
    if case["func"] != "none":
        g = g * _derivative(case["func"], gamma * xhat + beta)
    w = g * gamma
    error = ivar * (w - w.mean(1, keepdim=True) - xhat * (w * xhat).mean(1, keepdim=True))
    return {"error": error.view_as(delta), "dgamma": (g * xhat).sum(0), "dbeta": g.sum(0)}


def _through_8_bits(x):
    """What an activation is after it was kept in 8 bits: per group of 128 elements of a sample the lowest value, a step of
    1/255 of the range, and the number of steps of every element."""
    w, n = x.shape[0], x[0].numel()
    flat, short = x.reshape(w, n), -n % GROUP
    if short:
        flat = torch.cat([flat, flat[:, -1:].expand(w, short)], 1)
    flat = flat.view(w, -1, GROUP)
    low = flat.amin(2, keepdim=True)
    step = (flat.amax(2, keepdim=True) - low) * torch.tensor(1.0 / 255.0, device=x.device)
    step = torch.where(step < torch.finfo(torch.float32).tiny, 0.0, step)
    q = torch.where(step > 0, torch.round((flat - low) * (1.0 / step)), 0.0).clamp(0.0, 255.0)
    return (step * q + low).view(w, -1)[:, :n].reshape(x.shape)


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "pack":
        return {"out": _through_8_bits(s["x"])}
    if kind == "linear":
        x, delta = _through_8_bits(s["x"]).reshape(case["w"], -1), s["delta"].view(case["w"], -1)
        return {"dweight": torch.matmul(delta.t(), x), "dbias": delta.sum(0)}
    if kind == "back":
        return _backward(case, s["delta"], s["x"], s["gamma"], s["beta"], s["mean"], s["ivar"])
    out, mean, ivar = _forward(case, s["x"], s["gamma"], s["beta"])
    if kind == "norm":
        return {"out": out, "mean": mean, "ivar": ivar}
    return {"out": out, **_backward(case, s["delta"], _through_8_bits(s["x"]), s["gamma"], s["beta"], mean, ivar)}


def _run_own(s):
    mt = _bindings()
    case, t = s["case"], s["t"]
    kind = case["kind"]
    if kind == "pack":
        mt.CTensorMath.Pack(s["packed"], t["x"])
        mt.CTensorMath.Unpack(t["out"], s["packed"])
        return {"out": s["out"]}
    if kind == "linear":
        mt.CTensorMath.Pack(s["packed"], t["x"])
        mt.Fused.LinearBackwardWeightsSum(t["dweight"], t["dbias"], s["packed"], t["delta"], accumulate=False)
        return {"dweight": s["dweight"].view(case["out"], case["in"]), "dbias": s["dbias"].view(-1)}
    func = None if case["func"] == "none" else case["func"]
    out, (rows, n) = {}, _sizes(case)
    if kind != "back":
        mt.Fused.LayerNormForward(t["out"], t["x"], t["gamma"], t["beta"], t["mean"], t["ivar"], s.get("packed"), EPSILON, func)
        out["out"] = s["out"]
    if kind == "norm":
        return {"out": s["out"], "mean": s["mean"].view(rows, 1), "ivar": s["ivar"].view(rows, 1)}
    mt.Fused.LayerNormBackward(t["error"], t["dgamma"], t["dbeta"], t["delta"], t["gamma"], s["packed"] if kind == "step" else t["x"], t["mean"], t["ivar"],
                               beta=t["beta"], func=func, accumulate=False)
    out.update(error=s["error"], dgamma=s["dgamma"].view(n), dbeta=s["dbeta"].view(n))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- work and exact results ----------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "linear":
        b, n_in, n_out = case["w"], case["in"], case["out"]
        return {"bytes": 4.0 * (b * n_in + b * n_out + n_in * n_out + n_out), "flops": 2.0 * b * n_in * n_out}
    total = case["w"] * case["z"] * case["y"] * case["x"]
    if case["kind"] == "pack":
        return {"bytes": 8.0 * total, "flops": 6.0 * total}
    rows, n = _sizes(case)
    tensors, params, ops = {"norm": (2, 2, 8), "back": (3, 4, 12), "step": (4, 4, 24)}[case["kind"]]
    return {"bytes": 4.0 * (tensors * total + params * n + 2 * rows), "flops": float(ops * total)}


def _exact_8_bits(x):
    """The numbers that the 8-bit form stands for.  It holds the lowest value and the step of a group as 32-bit numbers, and
    the count of steps is decided on them; the sum is then taken in 64 bits."""
    w = x.shape[0]
    n = x.numel() // w
    out = torch.empty(w, n, dtype=torch.float64, device=x.device)
    whole = n // GROUP * GROUP
    for a, b, size in ((0, whole, GROUP), (whole, n, n - whole)):
        if a == b:
            continue
        part = x.reshape(w, n)[:, a:b].reshape(-1, size)
        low, high = part.min(1).values[:, None], part.max(1).values[:, None]
        step = (high - low) * torch.tensor(1.0 / 255.0, dtype=torch.float32, device=x.device)
        held = step >= 2.0 ** -126
        count = ((part - low) * step.reciprocal()).round().clamp(max=255)
        value = low.double() + step.double() * count.double()
        out[:, a:b] = torch.where(held, value, low.double()).view(w, -1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pack":
        return {"out": _exact_8_bits(s["x"]).view(s["x"].shape)}
    if kind == "linear":
        d = s["delta"].double().flatten(1)
        return {"dweight": d.T.contiguous() @ _exact_8_bits(s["x"]), "dbias": d.sum(0)}
    rows, n = _sizes(case)
    x, gamma, beta = s["x"].double().reshape(rows, n), s["gamma"].double().reshape(n), s["beta"].double().reshape(n)
    out = {}
    if kind == "back":
        mean, ivar = s["mean"].double().reshape(rows, 1), s["ivar"].double().reshape(rows, 1)
    else:
        mean = x.sum(1, keepdim=True) / n
        ivar = ((x - mean).pow(2).sum(1, keepdim=True) / n + EPSILON).rsqrt()
        y = (x - mean) * ivar * gamma + beta
        y = y.sigmoid() if case["func"] == "sigmoid" else y.tanh() if case["func"] == "tangence" else y
        out["out"] = y.view(s["x"].shape)
        if kind == "norm":
            return {**out, "mean": mean, "ivar": ivar}
        x = _exact_8_bits(s["x"]).reshape(rows, n)
    h = (x - mean) * ivar
    g = s["delta"].double().reshape(rows, n)
    pre = h * gamma + beta
    if case["func"] == "sigmoid":
        g = g * pre.sigmoid() * (-pre).sigmoid()
    elif case["func"] == "tangence":
        g = g / pre.cosh().pow(2)
    out["dgamma"], out["dbeta"] = (g * h).sum(0), g.sum(0)
    wg = g * gamma
    out["error"] = ((wg - wg.sum(1, keepdim=True) / n - h * ((wg * h).sum(1, keepdim=True) / n)) * ivar).view(s["delta"].shape)
    return out
