"""The measured cases of the layer operators (`vmc_pde_amd.layers`): the dense layer with its epilogue, layer norm, and clipping by the
global gradient norm.  `run` computes each in plain torch operations, or -- with `own` -- through the framework's entry points."""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32, "float64": torch.float64}
SIZE = {"bfloat16": 2, "float16": 2, "float32": 4, "float64": 8}
ACTIVATIONS = ("none", "tanh", "gelu", "silu")
EPS = 1e-6


def listed():
    return [
        # one token through the up projection of a wide block: bound by reading the weights once
        {"name": "dense_token", "op": "dense", "dtype": "bfloat16", "m": 1, "k": 4096, "n": 16384, "act": "silu", "bias": True, "residual": False,
         "scale": 1.0, "train": False, "kernel_t": False},
        # the same projection over a long prompt, the matrix pipe's largest case
        {"name": "dense_prompt", "op": "dense", "dtype": "bfloat16", "m": 8192, "k": 4096, "n": 16384, "act": "gelu", "bias": True, "residual": False,
         "scale": 1.0, "train": False, "kernel_t": False},
        # the down projection of a training step, residual added in the epilogue, with all its gradients
        {"name": "dense_train_bf16", "op": "dense", "dtype": "bfloat16", "m": 8192, "k": 8192, "n": 4096, "act": "gelu", "bias": True, "residual": True,
         "scale": 1.0, "train": True, "kernel_t": False},
        # a ragged batch, odd widths, the kernel stored transposed (out, in)
        {"name": "dense_ragged_f16", "op": "dense", "dtype": "float16", "m": 1537, "k": 1001, "n": 777, "act": "tanh", "bias": True, "residual": True,
         "scale": 0.5, "train": True, "kernel_t": True},
        # a conditioner wider than the flow kernels hold, in single precision, at the driver's 10 000 samples
        {"name": "dense_train_f32", "op": "dense", "dtype": "float32", "m": 10000, "k": 1024, "n": 1024, "act": "tanh", "bias": True, "residual": False,
         "scale": 1.0, "train": True, "kernel_t": False},
        # the headline flow's hidden layer (21 -> 21) over its 65 536 samples, 10 * tanh as the output layers have it
        {"name": "dense_train_f64", "op": "dense", "dtype": "float64", "m": 65536, "k": 21, "n": 21, "act": "tanh", "bias": True, "residual": False,
         "scale": 10.0, "train": True, "kernel_t": False},
        # one token's norm: latency
        {"name": "norm_token", "op": "norm", "dtype": "bfloat16", "weights": "float32", "rows": 1, "cols": 4096, "train": False},
        # the norm of a long training batch, weights kept in single precision
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bfloat16", "weights": "float32", "rows": 16384, "cols": 8192, "train": True},
        # odd width: no row but the first is aligned
        {"name": "norm_train_f32", "op": "norm", "dtype": "float32", "weights": "float32", "rows": 10000, "cols": 1001, "train": True},
        # narrow rows in the framework's own type, at the headline sample count
        {"name": "norm_train_f64", "op": "norm", "dtype": "float64", "weights": "float64", "rows": 65536, "cols": 21, "train": True},
        # the 51 leaves of the headline flow's parameter vector (4213 numbers): latency
        {"name": "clip_flow", "op": "clip", "dtype": "float64", "second": "float64", "tensors": 51, "total": 4213, "leaves": "flow", "factor": 0.5},
        # the gradients of a large model: matrices in bf16, vectors in f32
        {"name": "clip_large", "op": "clip", "dtype": "bfloat16", "second": "float32", "tensors": 290, "total": 500000000, "leaves": "spread", "factor": 0.3},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("dense", "dense", "norm", "clip"))
    if op == "dense":
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32", "float64"))
        train = rng.random() < 0.5
        most = {"bfloat16": 4e11, "float16": 4e11, "float32": 2e10, "float64": 1e10}[dtype]
        m, k, n = _log(rng, 1, 65536), _log(rng, 8, 16384), _log(rng, 8, 16384)
        while m * k * n > most / (3 if train else 1) or (m * k + k * n + m * n) * SIZE[dtype] > 2.5e8:
            if m >= k and m >= n:
                m = (m + 1) // 2
            elif k >= n:
                k = (k + 1) // 2
            else:
                n = (n + 1) // 2
        if rng.random() < 0.5:  # widths of networks are often, not always, multiples of eight
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        return {"op": "dense", "dtype": dtype, "m": m, "k": k, "n": n, "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.8,
                "residual": rng.random() < 0.5, "scale": rng.choice((1.0, 0.5, 10.0)), "train": train, "kernel_t": rng.random() < 0.3}
    if op == "norm":
        dtype = rng.choice(("bfloat16", "float16", "float32", "float64"))
        rows, cols = _log(rng, 1, 65536), _log(rng, 8, 16384)
        while rows * cols * SIZE[dtype] > 16384 * 8192 * 2:
            rows = (rows + 1) // 2
        weights = rng.choice((dtype, "float32")) if SIZE[dtype] == 2 else dtype
        return {"op": "norm", "dtype": dtype, "weights": weights, "rows": rows, "cols": cols, "train": rng.random() < 0.6}
    dtype = rng.choice(("bfloat16", "float16", "float32", "float64"))
    tensors = _log(rng, 1, 500)
    return {"op": "clip", "dtype": dtype, "second": rng.choice((dtype, "float32")), "tensors": tensors,
            "total": _log(rng, max(64, tensors), 800000000 // SIZE[dtype]), "leaves": "spread", "factor": rng.choice((0.01, 0.3, 0.9, 2.0))}


def _leaf_sizes(case):
    """(elements, whether it is of the first type) of each tensor of a clipping case."""
    if case["leaves"] == "flow":  # 4 blocks x 2 networks 1 -> 21 -> 21 -> 1 and the latent leaves, in the order of the flat vector
        return [(v, True) for v in [1, 2, 2] + [21, 21, 21, 441, 1, 21] * 8]
    count, total = case["tensors"], case["total"]
    weight = [1.0 if j % 4 else 0.0005 for j in range(count)]  # three matrices to a vector
    weight = [w * (1 + 0.6 * math.sin(1.7 * j)) for j, w in enumerate(weight)]
    sizes = [max(1, int(total * w / sum(weight))) for w in weight]
    return [(v, bool(j % 4) or count == 1) for j, v in enumerate(sizes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    wide = torch.float64 if case["dtype"] == "float64" else torch.float32

    def normal(*shape, scale=1.0, to=dtype):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=wide if to == torch.float64 or wide == torch.float32 else torch.float32)
        return t.mul_(scale).to(to)

    s = {"case": case}
    if case["op"] == "dense":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)
        s["kernel"] = normal(n, k, scale=k ** -0.5).t() if case["kernel_t"] else normal(k, n, scale=k ** -0.5)
        s["bias"] = normal(n, scale=0.2) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        s["dy"] = normal(m, n) if case["train"] else None
    elif case["op"] == "norm":
        rows, cols, weights = case["rows"], case["cols"], DTYPES[case["weights"]]
        channels = torch.exp(normal(cols, scale=0.5, to=wide))  # channels of unequal size about a row mean that is not zero
        s["x"] = (normal(rows, cols, to=wide).mul_(channels).add_(normal(rows, 1, to=wide))).to(dtype)
        s["weight"] = (normal(cols, scale=0.1, to=wide) + 1).to(weights)
        s["bias"] = normal(cols, scale=0.1, to=weights)
        s["dy"] = normal(rows, cols) if case["train"] else None
    else:
        leaves = _leaf_sizes(case)
        totals = [sum(v for v, first in leaves if first), sum(v for v, first in leaves if not first)]
        types = [dtype, DTYPES[case["second"]]]
        s["flat"] = [normal(t, scale=1e-3, to=ty) for t, ty in zip(totals, types) if t]
        s["out_flat"] = [torch.empty_like(t) for t in s["flat"]]
        at, s["grads"], s["out"] = [0, 0], [], []
        for v, first in leaves:  # the leaves lie behind each other in a flat vector of their type, as the framework's parameters do
            j = 0 if first else 1
            s["grads"].append(s["flat"][j][at[j]:at[j] + v])
            s["out"].append(s["out_flat"][j][at[j]:at[j] + v])
            at[j] += v
        s["max_norm"] = case["factor"] * 1e-3 * math.sqrt(sum(totals))
    return s


def _activate(z, act):
    """act(z) and act'(z)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    gate = 1 / (1 + torch.exp(-z))
    return z * gate, gate * (1 + z * (1 - gate))


def _plain_dense(s, c):
    to = s["x"].dtype
    wide = torch.float64 if to == torch.float64 else torch.float32
    x, kernel = s["x"].to(wide), s["kernel"].to(wide)
    z = x @ kernel
    if c["bias"]:
        z = z + s["bias"].to(wide)
    a, slope = _activate(z, c["act"])
    y = c["scale"] * a
    if c["residual"]:
        y = y + s["residual"].to(wide)
    out = {"y": y.to(to)}
    if c["train"]:
        dz = c["scale"] * slope * s["dy"].to(wide)
        out["dx"], out["dkernel"] = (dz @ kernel.t()).to(to), (x.t() @ dz).to(to)
        if c["bias"]:
            out["dbias"] = dz.sum(0).to(to)
    return out


def _plain_norm(s, c):
    to, weights = s["x"].dtype, s["weight"].dtype
    wide = torch.float64 if to == torch.float64 else torch.float32
    x, w, b = s["x"].to(wide), s["weight"].to(wide), s["bias"].to(wide)
    centred = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    h = centred * rstd
    out = {"y": (h * w + b).to(to)}
    if c["train"]:
        dy = s["dy"].to(wide)
        g = dy * w
        out["dx"] = (rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))).to(to)
        out["dweight"], out["dbias"] = (dy * h).sum(0).to(weights), dy.sum(0).to(weights)
    return out


def _plain_clip(s, c):
    norm = torch.sqrt(torch.stack([torch.sum(t.double().square()) for t in s["flat"]]).sum())
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
    wide = [t if t.dtype == torch.float64 else t.float() for t in s["flat"]]
    return {"norm": norm, "grads": [(w * factor.to(w.dtype)).to(t.dtype) for w, t in zip(wide, s["flat"])]}


def run(state):
    c = state["case"]
    if own:
        from vmc_pde_amd import layers
        if c["op"] == "dense":
            x, kernel, bias, more = state["x"], state["kernel"], state["bias"], dict(activation=c["act"], scale=c["scale"], residual=state["residual"])
            if not c["train"]:
                return {"y": layers.dense(x, kernel, bias, **more)}
            y, slope = layers.dense(x, kernel, bias, want_slope=True, **more)
            dx, dkernel, dbias = layers.dense_backward(state["dy"], x, kernel, slope, scale=c["scale"], want_bias=c["bias"])
            out = {"y": y, "dx": dx, "dkernel": dkernel}
            return {**out, "dbias": dbias} if c["bias"] else out
        if c["op"] == "norm":
            if not c["train"]:
                return {"y": layers.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS)}
            y, mean, rstd = layers.layer_norm(state["x"], state["weight"], state["bias"], eps=EPS, want_stats=True)
            dx, dweight, dbias = layers.layer_norm_backward(state["dy"], state["x"], mean, rstd, state["weight"])
            return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
        norm = layers.clip_by_global_norm(state["grads"], state["max_norm"], out=state["out"])
        return {"norm": norm, "grads": state["out_flat"]}
    return {"dense": _plain_dense, "norm": _plain_norm, "clip": _plain_clip}[c["op"]](state, c)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "dense":
        m, k, n = case["m"], case["k"], case["n"]
        moved = m * k + k * n + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        if case["train"]:
            moved += m * n + m * k + k * n + (n if case["bias"] else 0)
        return {"bytes": size * moved, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    if case["op"] == "norm":
        cells, cols, weights = case["rows"] * case["cols"], case["cols"], SIZE[case["weights"]]
        if case["train"]:
            return {"bytes": 4 * cells * size + 4 * cols * weights, "flops": 20 * cells}
        return {"bytes": 2 * cells * size + 2 * cols * weights, "flops": 8 * cells}
    sizes = [(v, SIZE[case["dtype"] if first else case["second"]]) for v, first in _leaf_sizes(case)]
    return {"bytes": 2 * sum(v * b for v, b in sizes) + 8, "flops": 3 * sum(v for v, _ in sizes)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        grads = [t.to(torch.float64) for t in s["flat"]]
        norm = math.sqrt(math.fsum(float(torch.dot(t, t)) for t in grads))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [t * min(1.0, s["max_norm"] / norm) for t in grads]}
    # the definitions in 64 bits; the gradients by automatic differentiation of them
    with torch.enable_grad():
        leaf = {name: s[name].detach().to(torch.float64).requires_grad_(case["train"]) for name in ("x", "kernel", "weight", "bias") if s.get(name) is not None}
        if case["op"] == "dense":
            z = torch.mm(leaf["x"], leaf["kernel"])
            z = torch.add(z, leaf["bias"]) if case["bias"] else z
            act = {"none": lambda v: v, "tanh": torch.tanh, "gelu": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2)),
                   "silu": lambda v: v / (1 + torch.exp(-v))}[case["act"]]
            y = act(z).mul(case["scale"])
            y = y + s["residual"].to(torch.float64) if case["residual"] else y
            names = {"dx": "x", "dkernel": "kernel"} | ({"dbias": "bias"} if case["bias"] else {})
        else:
            x = leaf["x"]
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            y = (x - mean) * torch.rsqrt(var + EPS) * leaf["weight"] + leaf["bias"]
            names = {"dx": "x", "dweight": "weight", "dbias": "bias"}
        out = {"y": y.detach()}
        if case["train"]:
            found = torch.autograd.grad(y, [leaf[v] for v in names.values()], s["dy"].to(torch.float64))
            out.update(zip(names, found))
    return out
