"""The layer operators (vmc_pde_amd.layers) against their plain 64-bit forms, with bounds counted in roundings (tests/helpers_layers.py)."""
import math

import pytest
import torch

import helpers_layers as plain

pytestmark = pytest.mark.gpu
DTYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]
IDS = ["f64", "f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def layers():
    from vmc_pde_amd import layers as module
    return module


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, dtype=torch.float64)).to(dtype).cuda()


# ---- dense -------------------------------------------------------------------------------------------------------------------------------

SIZES = [(0, 5, 7), (1, 1, 1), (1, 8, 16), (3, 5, 7), (17, 33, 65), (33, 64, 8), (128, 128, 128), (130, 129, 131), (257, 64, 40), (1, 2048, 264), (5, 1000, 513),
         (64, 520, 24), (1000, 21, 21), (2049, 40, 9), (300, 520, 264), (512, 256, 512), (40, 16, 1300), (3500, 72, 4100), (40, 3601, 3700), (70, 32, 32), (70, 33, 32), (333, 8, 17), (333, 16, 16), (17, 17, 1), (9000, 24, 30), (200, 1, 21), (700, 43, 43), (520, 48, 30), (1000, 12, 48), (90, 40, 7), (64, 49, 48)]
ACTS = ["none", "tanh", "gelu", "silu"]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("number, size", list(enumerate(SIZES)), ids=["x".join(map(str, s)) for s in SIZES])
def test_dense_and_its_gradients(layers, dtype, number, size):
    rows, n_in, n_out = size
    act, scale = ACTS[(number + DTYPES.index(dtype)) % 4], (1.0, 10.0, -0.5)[number % 3]
    x = normal((rows, n_in), dtype, 10 * number)
    transposed = number % 3 == 1
    kernel = normal((n_out, n_in) if transposed else (n_in, n_out), dtype, 10 * number + 1, n_in ** -0.5)
    kernel = kernel.t() if transposed else kernel
    bias = normal((n_out,), dtype, 10 * number + 2, 0.3) if number % 4 != 1 else None
    residual = normal((rows, n_out), dtype, 10 * number + 3) if number % 2 else None
    dy = normal((rows, n_out), dtype, 10 * number + 4)
    y, slope = layers.dense(x, kernel, bias, activation=act, scale=scale, residual=residual, want_slope=True)
    dx, dkernel, dbias = layers.dense_backward(dy, x, kernel, slope, scale=scale)
    want = plain.dense(x, kernel, bias, residual, act, scale, dy, dtype)
    assert (slope is None) == (act == "none")
    for name, got in (("y", y), ("slope", slope), ("dx", dx), ("dkernel", dkernel), ("dbias", dbias)):
        if got is not None:
            plain.agrees(got, want[name], name)
    if rows * n_out >= 64:
        for name, got in (("dx", dx), ("dkernel", dkernel)):       # roundings of dz and of the output, and of fp32 / fp64 sums
            plain.near(got, want[name], 3 if dtype in (torch.float16, torch.bfloat16) else 40, dtype, name)
    alone = layers.dense(x, kernel, bias, activation=act, scale=scale, residual=residual)
    assert torch.equal(alone, y)
    again = layers.dense_backward(dy, x, kernel, slope, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dkernel, dbias)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dense_gradients_one_at_a_time(layers, dtype):
    x, kernel, dy = normal((70, 24), dtype, 1), normal((24, 40), dtype, 2, 0.2), normal((70, 40), dtype, 3)
    _, slope = layers.dense(x, kernel, activation="gelu", want_slope=True)
    whole = layers.dense_backward(dy, x, kernel, slope, scale=2.0)
    for k, name in enumerate(("want_x", "want_kernel", "want_bias")):
        flags = {n: n == name for n in ("want_x", "want_kernel", "want_bias")}
        only = layers.dense_backward(dy, x, kernel, slope, scale=2.0, **flags)
        assert torch.equal(only[k], whole[k]) and all(v is None for j, v in enumerate(only) if j != k)
    assert layers.dense_backward(dy, x, kernel, slope, want_x=False, want_kernel=False, want_bias=False) == (None, None, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dense_takes_views(layers, dtype):
    """Row pitches, an odd offset into a flat vector, leading axes, an expanded row, every other column: as their contiguous copies."""
    flat = normal((4000,), dtype, 5)
    wide = normal((2, 50, 90), dtype, 6)
    kernel = flat[3:3 + 31 * 45].view(31, 45)
    bias = flat[1999:1999 + 45]
    for x in (wide[..., 7:38], wide[0, :, 1:32], wide[:, ::2, 2:33], wide[..., 4:66:2], wide[0, 0, 10:41].expand(6, 31), wide.transpose(0, 1)[..., 0:31], wide[1, 3, 5:36]):
        residual = normal((*x.shape[:-1], 60), dtype, 7)[..., 3:48]
        y, slope = layers.dense(x, kernel, bias, activation="tanh", residual=residual, want_slope=True)
        clean = layers.dense(x.contiguous(), kernel.clone(), bias.clone(), activation="tanh", residual=residual.contiguous(), want_slope=True)
        assert y.shape == (*x.shape[:-1], 45) and torch.equal(y, clean[0]) and torch.equal(slope, clean[1])
        dy = normal((*x.shape[:-1], 61), dtype, 8)[..., 1:46]
        got = layers.dense_backward(dy, x, kernel, slope)
        want = layers.dense_backward(dy.contiguous(), x.contiguous(), kernel.clone(), slope)
        assert got[0].shape == x.shape and all(torch.equal(a, b) for a, b in zip(got, want))
    for odd in (normal((31, 100), dtype, 9)[:, 3:48], normal((45, 80), dtype, 10)[:, 5:36].t(), normal((62, 90), dtype, 11)[::2, ::2]):
        x, dy = wide[0, :, :31], normal((50, 45), dtype, 12)
        assert torch.equal(layers.dense(x, odd), layers.dense(x, odd.t().contiguous().t() if odd.stride(0) == 1 else odd.contiguous()))
        got, want = layers.dense_backward(dy, x, odd), plain.dense(x, odd, None, None, "none", 1.0, dy, dtype)
        for name, g in zip(("dx", "dkernel", "dbias"), got):
            plain.agrees(g, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 8])
def test_dense_of_few_rows(layers, dtype, rows):
    """A token or a handful of them, either layout, odd widths and pitches, with and without slices of k: the forward pass and dx."""
    for number, (n_in, n_out) in enumerate([(1, 8), (7, 9), (63, 65), (64, 200), (129, 71), (515, 1003), (5000, 40), (9001, 50), (2100, 17)]):
        act, scale = ACTS[(number + rows) % 4], (1.0, 10.0, -0.5)[number % 3]
        x, dy = normal((rows, n_in + 1), dtype, 10 * number)[:, 1:], normal((rows, n_out + 3), dtype, 10 * number + 4)[:, 2:2 + n_out]
        bias, residual = normal((n_out,), dtype, 10 * number + 2, 0.3), normal((rows, n_out), dtype, 10 * number + 3) if number % 2 else None
        for kernel in (normal((n_in, n_out + number % 3), dtype, 10 * number + 1, n_in ** -0.5)[:, number % 3:],
                       normal((n_out, n_in + number % 2), dtype, 10 * number + 5, n_in ** -0.5)[:, number % 2:].t()):
            y, slope = layers.dense(x, kernel, bias, activation=act, scale=scale, residual=residual, want_slope=True)
            dx, _, _ = layers.dense_backward(dy, x, kernel, slope, scale=scale, want_kernel=False, want_bias=False)
            want = plain.dense(x, kernel, bias, residual, act, scale, dy, dtype)
            for name, got in (("y", y), ("slope", slope), ("dx", dx)):
                if got is not None:
                    plain.agrees(got, want[name], name)
            if rows * n_in >= 64:
                plain.near(dx, want["dx"], 3 if dtype in (torch.float16, torch.bfloat16) else 40, dtype, "dx")
            assert torch.equal(layers.dense(x.contiguous(), kernel.clone(), bias, activation=act, scale=scale, residual=residual), y)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("across", [0, 1])
@pytest.mark.parametrize("rows", [3, 37])
def test_dense_writes_its_rows_only(layers, dtype, across, rows):
    """A target with a row pitch: what lies between and behind the rows stays as it was."""
    from vmc_pde_amd import _native as nat
    n_in, n_out, pitch = 72, 43, 56
    x, kernel = normal((rows, n_in), dtype, 1), normal((n_out, n_in) if across else (n_in, n_out), dtype, 2, 0.1)
    y = torch.full((rows + 3, pitch), -7.0, dtype=dtype, device="cuda")
    a = nat.DenseArgs(layers.DTYPE[dtype], 2, across, 0, rows, n_in, n_out, x.data_ptr(), n_in, kernel.data_ptr(), n_in if across else n_out, None, None, 0, 1.0,
                      y.data_ptr(), pitch)
    need = nat.lib().vmcpde_dense_workspace_bytes(a, 0)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    nat.call("vmcpde_dense", a, ws.data_ptr(), need, nat.stream())
    assert torch.equal(y[:rows, :n_out], layers.dense(x, kernel.t() if across else kernel, activation="gelu"))
    assert bool((y[rows:] == -7).all()) and bool((y[:, n_out:] == -7).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dense_keeps_what_is_not_finite_in_its_row(layers, dtype):
    """Infinities and NaN reach their own row of y and dx, and nothing else; what lies behind a view's columns reaches nothing."""
    whole = torch.full((40, 320), float("nan"), dtype=dtype, device="cuda")
    kernel = torch.full((304, 80), float("nan"), dtype=dtype, device="cuda")
    for width in (304, 301, 130, 48, 45, 7):
        whole[:, :width], kernel[:width, :52] = normal((40, width), dtype, 1), normal((width, 52), dtype, 2, 0.2)
        whole[:, width:], kernel[width:] = float("nan"), float("nan")
        x, k = whole[:, :width].clone(), kernel[:width, :52]
        clean = layers.dense(whole[:, :width], k, activation="silu")
        assert bool(torch.isfinite(clean).all())
        x[7, 3], x[11, 5], x[20, 0] = float("nan"), float("inf"), -float("inf")
        y, slope = layers.dense(x, k, activation="gelu", want_slope=True)
        reference = layers.dense(whole[:, :width], k, activation="gelu")
        fine = [r for r in range(40) if r not in (7, 11, 20)]
        assert torch.equal(y[fine], reference[fine]) and bool(torch.isnan(y[7]).all())
        z = x[11].double() @ k.double()
        assert torch.equal(torch.isinf(y[11]), torch.isposinf(z)) and not bool(torch.isnan(y[11]).any()) and not bool(torch.isnan(slope[[11, 20]]).any())
        assert bool((y[11][torch.isneginf(z)] == 0).all()) and bool((slope[11][torch.isposinf(z)] == 1).all())
        dy = normal((40, 52), dtype, 3)
        dy[4, 1] = float("nan")
        dx, _, dbias = layers.dense_backward(dy, whole[:, :width], k)
        assert bool(torch.isnan(dx[4]).all()) and bool(torch.isfinite(dx[:4]).all()) and bool(torch.isfinite(dx[5:]).all())
        assert bool(torch.isnan(dbias[1])) and int(torch.isnan(dbias).sum()) == 1


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_activations_over_their_whole_range(layers, dtype, act):
    z = torch.cat([torch.linspace(-30, 30, 4001, dtype=torch.float64), torch.logspace(-9, 4, 500, dtype=torch.float64), -torch.logspace(-9, 4, 500, dtype=torch.float64)])
    x = z.to(dtype).cuda()[:, None]
    y, slope = layers.dense(x, torch.ones(1, 1, dtype=dtype, device="cuda"), activation=act, want_slope=True)
    want = plain.dense(x, torch.ones(1, 1, dtype=dtype), None, None, act, 1.0, None, dtype)
    plain.agrees(y, want["y"], "y")
    plain.agrees(slope, want["slope"], "slope")


@pytest.mark.parametrize("act", ACTS)
def test_dense_gradients_against_differences(layers, act):
    x, kernel, bias, dy = normal((9, 7), torch.float64, 1), normal((7, 5), torch.float64, 2), normal((5,), torch.float64, 3), normal((9, 5), torch.float64, 4)
    _, slope = layers.dense(x, kernel, bias, activation=act, scale=1.7, want_slope=True)
    grads = layers.dense_backward(dy, x, kernel, slope, scale=1.7)
    # central differences: h^2 |f'''| / 6 ~ 1e-10 and 2^-53 |f| / h ~ 1e-10, a hundredfold of both
    h = 1e-5
    for t, grad in zip((x, kernel, bias), grads):
        for at in range(0, t.numel(), 3):
            old = float(t.view(-1)[at])
            f = []
            for step in (h, -h):
                t.view(-1)[at] = old + step
                f.append(float((layers.dense(x, kernel, bias, activation=act, scale=1.7) * dy).sum()))
            t.view(-1)[at] = old
            assert abs((f[0] - f[1]) / (2 * h) - float(grad.view(-1)[at])) < 2e-8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 70000, 5), (70000, 6, 10), (4, 9, 70001)])
def test_dense_long_axes(layers, dtype, size):
    """One axis far longer than a tile: long sums, many rows, many columns."""
    rows, n_in, n_out = size
    x, kernel, dy = normal((rows, n_in), dtype, 1), normal((n_in, n_out), dtype, 2, n_in ** -0.5), normal((rows, n_out), dtype, 3)
    y, slope = layers.dense(x, kernel, activation="tanh", want_slope=True)
    grads = layers.dense_backward(dy, x, kernel, slope)
    want = plain.dense(x, kernel, None, None, "tanh", 1.0, dy, dtype)
    plain.agrees(y, want["y"], "y")
    for name, got in zip(("dx", "dkernel", "dbias"), grads):
        plain.agrees(got, want[name], name)
        plain.near(got, want[name], 3 if dtype == torch.bfloat16 else 100, dtype, name)


def test_dense_beyond_32_bits(layers):
    """An operand whose last rows lie more than 2^32 bytes behind its first ones."""
    rows, n = 8400, 262144
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    x[-40:, -40:] = normal((40, 40), torch.bfloat16, 1)
    kernel = torch.zeros((n, 8), dtype=torch.bfloat16, device="cuda")
    kernel[-40:] = normal((40, 8), torch.bfloat16, 2)
    y = layers.dense(x, kernel)
    want = plain.dense(x[-40:, -40:], kernel[-40:], None, None, "none", 1.0, None, torch.bfloat16)["y"]
    plain.agrees(y[-40:], want, "y")
    assert not bool(y[:-40].any())
    dy = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    dy[-40:] = normal((40, 8), torch.bfloat16, 3)
    _, dkernel, _ = layers.dense_backward(dy, x, kernel, want_x=False)
    want = plain.dense(x[-40:, -40:], kernel[-40:], None, None, "none", 1.0, dy[-40:], torch.bfloat16)["dkernel"]
    plain.agrees(dkernel[-40:], want, "dkernel")
    assert not bool(dkernel[:-40].any())


def test_dense_of_a_token_beyond_32_bits(layers):
    """One row, whose kernel's last lines lie more than 2^32 bytes behind its first ones: across k (the product) and along it (dx)."""
    n_in, n_out = 8400, 262144
    x = torch.zeros((1, n_in), dtype=torch.bfloat16, device="cuda")
    x[:, -40:] = normal((1, 40), torch.bfloat16, 1)
    dy = torch.zeros((1, n_out), dtype=torch.bfloat16, device="cuda")
    dy[:, -40:] = normal((1, 40), torch.bfloat16, 2)
    kernel = torch.zeros((n_in, n_out), dtype=torch.bfloat16, device="cuda")
    kernel[-40:, -40:] = normal((40, 40), torch.bfloat16, 3)
    want = plain.dense(x[:, -40:], kernel[-40:, -40:], None, None, "none", 1.0, dy[:, -40:], torch.bfloat16)
    y = layers.dense(x, kernel)
    dx, _, _ = layers.dense_backward(dy, x, kernel, want_kernel=False, want_bias=False)
    for name, got in (("y", y), ("dx", dx)):
        plain.agrees(got[:, -40:], want[name], name)
        assert not bool(got[:, :-40].any())


def test_dense_refuses_shapes(layers):
    x, k = torch.zeros(3, 4, device="cuda"), torch.zeros(4, 5, device="cuda")
    for call in (lambda: layers.dense(x, torch.zeros(5, 4, device="cuda")), lambda: layers.dense(x, k, torch.zeros(4, device="cuda")),
                 lambda: layers.dense(x, k, residual=torch.zeros(3, 4, device="cuda")), lambda: layers.dense(x, k, activation="relu"),
                 lambda: layers.dense(x[0, 0], k), lambda: layers.dense(x[:, :0], k[:0]), lambda: layers.dense(x, k[0]), lambda: layers.dense(x, k, torch.zeros(5)),
                 lambda: layers.dense_backward(torch.zeros(3, 4, device="cuda"), x, k), lambda: layers.dense_backward(torch.zeros(2, 5, device="cuda"), x, k),
                 lambda: layers.dense_backward(torch.zeros(3, 5, device="cuda"), x, k, torch.zeros(3, 4, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: layers.dense(x, k.half()), lambda: layers.dense_backward(torch.zeros(3, 5, device="cuda"), x, k, torch.zeros(3, 5, device="cuda").double()),
                 lambda: layers.dense_backward(torch.zeros(3, 5, device="cuda").half(), x, k)):
        with pytest.raises(TypeError):
            call()
    from vmc_pde_amd import _native as nat
    with pytest.raises(nat.VmcpdeError, match="scale"):
        layers.dense(x, k, scale=float("nan"))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_native_calls_and_python_agree(layers, dtype, monkeypatch):
    """Both forms of every operator on plain tensors, views, parameters, no rows, one axis, negated views and whole numbers for floats: the same bits."""
    from vmc_pde_amd import _native as nat
    wide, flat = normal((3, 9, 40), dtype, 1), normal((900,), dtype, 2)
    kernel, bias = normal((24, 17), dtype, 3, 0.2), flat[1:18]
    views = [wide[..., 3:27], wide[1, :, :24], wide[:, ::2, 16:40], wide[0, 0, :24], wide.transpose(0, 1)[..., :24], wide[..., ::2][..., :20].repeat(1, 1, 2)[..., :24],
             wide[:0, :, :24], torch.nn.Parameter(wide[0, :, :24].contiguous()), torch._neg_view(wide[0, :, :24].contiguous()), wide[2, :1, 2:26]]
    kernels = [kernel, kernel.t().contiguous().t(), torch._neg_view(kernel), torch.nn.Parameter(kernel), normal((48, 34), dtype, 4)[::2, ::2]]

    def everything():
        for x in views:
            for k in kernels:
                residual = wide.new_ones((*x.shape[:-1], 17))
                y, slope = layers.dense(x, k, bias, activation="gelu", scale=2, residual=residual, want_slope=True)
                yield from (y, slope, layers.dense(x, k), *layers.dense_backward(y, x, k, slope, scale=2), *layers.dense_backward(y, x, k, want_x=False))
            w, b = flat[5:29], torch._neg_view(flat[100:124])
            y, mean, rstd = layers.layer_norm(x, w, b, eps=1, want_stats=True)
            yield from (y, mean, rstd, layers.layer_norm(x, bias=w), *layers.layer_norm_backward(y, x, mean, rstd, w), *layers.layer_norm_backward(y, x, mean, rstd, want_bias=False))
            copies = [x.detach().clone(), kernel.clone()]
            yield from (layers.clip_by_global_norm(copies, 1), *copies, layers.global_norm([x, kernel.contiguous()]) if x.is_contiguous() else None)

    with torch.no_grad():
        native = list(everything())
        monkeypatch.setattr(nat, "_calls", (None,))
        for a, b in zip(native, everything()):
            assert (a is None) == (b is None)
            assert a is None or a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)
    positive, negative = layers.dense(wide[0, :, :24], kernel), layers.dense(views[8], kernel)
    assert torch.equal(positive, -negative)


# ---- layer norm --------------------------------------------------------------------------------------------------------------------------

NORM_SIZES = [(0, 5), (1, 1), (3, 1), (5, 2), (65, 21), (33, 64), (7, 100), (300, 129), (17, 512), (40, 777), (9, 1025), (66, 2048), (3, 4096), (600, 4099), (5, 8192),
              (2, 10001), (3, 16384), (2, 33000), (700, 70), (2050, 8), (3, 20001), (3, 32768), (5, 40003)]


@pytest.mark.parametrize("dtype, weights", [(d, d) for d in DTYPES] + [(torch.float16, torch.float32), (torch.bfloat16, torch.float32)],
                         ids=IDS + ["f16-f32", "bf16-f32"])
@pytest.mark.parametrize("number, size", list(enumerate(NORM_SIZES)), ids=["x".join(map(str, s)) for s in NORM_SIZES])
def test_layer_norm_and_its_gradients(layers, dtype, weights, number, size):
    rows, cols = size
    x = (normal((rows, cols), torch.float64, number) + 3 * normal((rows, 1), torch.float64, number + 100)).to(dtype)
    weight = normal((cols,), weights, number + 200, 0.3) + 1 if number % 3 != 2 else None
    bias = normal((cols,), weights, number + 300) if number % 2 == 0 and (weight is not None or weights == dtype) else None
    dy = normal((rows, cols), dtype, number + 400)
    y, mean, rstd = layers.layer_norm(x, weight, bias, eps=1e-5, want_stats=True)
    grads = layers.layer_norm_backward(dy, x, mean, rstd, weight, weight_dtype=None if weight is not None else weights)
    want = plain.layer_norm(x, weight, bias, 1e-5, dy, dtype, weights)
    for name, got in (("y", y), ("mean", mean), ("rstd", rstd), ("dx", grads[0]), ("dweight", grads[1]), ("dbias", grads[2])):
        plain.agrees(got, want[name], name)
    assert grads[1].dtype == weights
    assert torch.equal(layers.layer_norm(x, weight, bias, eps=1e-5), y)
    for k in range(3):
        only = layers.layer_norm_backward(dy, x, mean, rstd, weight, want_x=k == 0, want_weight=k == 1, want_bias=k == 2,
                                          weight_dtype=None if weight is not None else weights)
        assert torch.equal(only[k], grads[k]) and sum(v is not None for v in only) == 1


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [37, 1000])
def test_layer_norm_takes_views(layers, dtype, cols):
    flat = normal((4 * cols + 9,), dtype, 1)
    wide = normal((2, 20, cols + 13), dtype, 2)
    weight, bias = flat[1:1 + cols], flat[cols + 3:2 * cols + 3]
    for x in (wide[..., 3:3 + cols], wide[:, ::3, 1:1 + cols], wide[0, 4, 5:5 + cols], wide[0, 0, :cols].expand(4, cols), wide.transpose(0, 1)[..., :cols]):
        y, mean, rstd = layers.layer_norm(x, weight, bias, want_stats=True)
        assert y.shape == x.shape and mean.shape == x.shape[:-1]
        assert torch.equal(y, layers.layer_norm(x.contiguous(), weight.clone(), bias.clone()))
        dy = normal((*x.shape[:-1], cols + 3), dtype, 3)[..., 2:2 + cols]
        got = layers.layer_norm_backward(dy, x, mean, rstd, weight)
        want = layers.layer_norm_backward(dy.contiguous(), x.contiguous(), mean, rstd, weight.clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [21, 1000, 5000])
def test_layer_norm_of_difficult_rows(layers, dtype, cols):
    """Constant rows (no variance), rows far from zero, infinities and NaN: each stays in its row."""
    x = normal((12, cols), dtype, 1)
    x[3] = 2.5
    x[5] = 0
    y, mean, rstd = layers.layer_norm(x, eps=1e-6, want_stats=True)
    assert not bool(y[3].any()) and not bool(y[5].any())        # deviations of equal elements are exact zeros
    dy = normal((12, cols), dtype, 2)
    clean = layers.layer_norm_backward(dy, x, mean, rstd)
    assert all(bool(torch.isfinite(g).all()) for g in clean)
    x[7, cols // 2], x[9, 1] = float("nan"), float("inf")
    bad, bad_mean, bad_rstd = layers.layer_norm(x, want_stats=True)
    fine = [r for r in range(12) if r not in (7, 9)]
    assert torch.equal(bad[fine], y[fine]) and bool(torch.isnan(bad[7]).all()) and bool(torch.isnan(bad[9]).any())
    dx, _, _ = layers.layer_norm_backward(dy, x, bad_mean, bad_rstd)
    assert torch.equal(dx[fine], clean[0][fine])
    if dtype in (torch.float64, torch.float32):
        far = normal((4, cols), torch.float64, 3) + (1e6 if dtype == torch.float64 else 300.0)
        far = far.to(dtype)
        plain.agrees(layers.layer_norm(far, eps=0.0), plain.layer_norm(far, None, None, 0.0, None, dtype, dtype)["y"], "y")


def test_layer_norm_gradients_against_differences(layers):
    x, weight, bias, dy = normal((4, 9), torch.float64, 1), normal((9,), torch.float64, 2), normal((9,), torch.float64, 3), normal((4, 9), torch.float64, 4)
    _, mean, rstd = layers.layer_norm(x, weight, bias, want_stats=True)
    h = 1e-5
    for t, grad in zip((x, weight, bias), layers.layer_norm_backward(dy, x, mean, rstd, weight)):
        for at in range(t.numel()):
            old, f = float(t.view(-1)[at]), []
            for step in (h, -h):
                t.view(-1)[at] = old + step
                f.append(float((layers.layer_norm(x, weight, bias) * dy).sum()))
            t.view(-1)[at] = old
            assert abs((f[0] - f[1]) / (2 * h) - float(grad.view(-1)[at])) < 5e-8       # (as for the dense layer; third derivatives are a few times larger)


def test_layer_norm_beyond_32_bits(layers):
    x = torch.empty((300000, 8192), dtype=torch.bfloat16, device="cuda")
    x[-3:] = normal((3, 8192), torch.bfloat16, 1)
    x[:-3] = normal((1, 8192), torch.bfloat16, 2)
    y, mean, rstd = layers.layer_norm(x, want_stats=True)
    plain.agrees(y[-3:], plain.layer_norm(x[-3:], None, None, 1e-6, None, torch.bfloat16, torch.bfloat16)["y"], "y")
    assert torch.equal(y[0].expand(5, 8192), y[-8:-3])
    dx, _, _ = layers.layer_norm_backward(y, x, mean, rstd, want_weight=False, want_bias=False)
    assert torch.equal(dx[0].expand(5, 8192), dx[-8:-3])


@pytest.mark.parametrize("dtype, weights, size", [(torch.bfloat16, torch.float32, (4500000, 3)), (torch.float64, torch.float64, (3001, 1)), (torch.float32, torch.float32, (70001, 3)),
                                                  (torch.float16, torch.float16, (257, 7)), (torch.bfloat16, torch.bfloat16, (1025, 4))],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
def test_layer_norm_of_rows_shorter_than_a_vector(layers, dtype, weights, size):
    rows, cols = size
    x, dy = normal((rows, cols + 2), dtype, 1)[:, 1:1 + cols], normal((rows, cols + 1), dtype, 2)[:, :cols]
    weight, bias = normal((cols,), weights, 3), normal((cols,), weights, 4)
    y, mean, rstd = layers.layer_norm(x, weight, bias, eps=1e-3, want_stats=True)
    grads = layers.layer_norm_backward(dy, x, mean, rstd, weight)
    want = plain.layer_norm(x, weight, bias, 1e-3, dy, dtype, weights)
    for name, got in (("y", y), ("mean", mean), ("rstd", rstd), ("dx", grads[0]), ("dweight", grads[1]), ("dbias", grads[2])):
        plain.agrees(got, want[name], name)
    for k in range(3):
        only = layers.layer_norm_backward(dy, x, mean, rstd, weight, want_x=k == 0, want_weight=k == 1, want_bias=k == 2)
        assert torch.equal(only[k], grads[k])


def test_layer_norm_refuses_shapes(layers):
    x = torch.zeros(3, 4, device="cuda")
    stats = torch.zeros(3, device="cuda")
    for call in (lambda: layers.layer_norm(x, torch.zeros(3, device="cuda")), lambda: layers.layer_norm(x[0, 0]), lambda: layers.layer_norm(x[:, :0]),
                 lambda: layers.layer_norm(x, eps=-1.0), lambda: layers.layer_norm(x, torch.zeros(4)), lambda: layers.layer_norm_backward(x[:2], x, stats, stats),
                 lambda: layers.layer_norm_backward(x, x, stats[:2], stats)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: layers.layer_norm(x, torch.zeros(4, device="cuda").half()), lambda: layers.layer_norm(x.half(), torch.zeros(4, device="cuda").double()),
                 lambda: layers.layer_norm(x.half(), torch.zeros(4, device="cuda").half(), torch.zeros(4, device="cuda")),
                 lambda: layers.layer_norm_backward(x, x, stats.double(), stats), lambda: layers.layer_norm_backward(x, x.half(), stats, stats),
                 lambda: layers.layer_norm_backward(x, x, stats, stats, weight_dtype=torch.bfloat16)):
        with pytest.raises(TypeError):
            call()


# ---- global norm -------------------------------------------------------------------------------------------------------------------------

def parts(total_sizes, dtypes, seed):
    """Tensors of the given sizes, some of them views at odd offsets of a flat vector."""
    out = []
    for k, n in enumerate(total_sizes):
        dtype = dtypes[k % len(dtypes)]
        flat = normal((n + 5,), dtype, seed + k, 0.1 * (1 + k % 7))
        out.append(flat[k % 4:k % 4 + n])
    return out


@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES], ids=IDS + ["mixed"])
@pytest.mark.parametrize("sizes", [[1], [0, 3, 0], [21, 21, 441, 1, 2], [4213], [32768], [32769], [100003, 7, 0, 8192, 65537], [50] * 300, [9000, 3] * 120],
                         ids=["1", "0-3-0", "leaves", "4213", "32768", "32769", "long", "300", "240"])
def test_clip_by_global_norm(layers, dtypes, sizes):
    tensors = parts(sizes, dtypes, 7)
    before = [t.clone() for t in tensors]
    want = math.sqrt(math.fsum(float((t.double().cpu() ** 2).sum()) for t in tensors))
    norm = layers.global_norm(tensors)
    assert norm.dtype == torch.float64 and norm.dim() == 0
    assert abs(float(norm) - want) <= 1e-12 * want           # some 1e4 additions of positive numbers in fp64, each within 2^-53
    for factor in (0.37, 1.5):
        out = [torch.full_like(t, -1) for t in tensors]
        got = layers.clip_by_global_norm(tensors, factor * want, out=out)
        assert torch.equal(got, norm) and all(torch.equal(a, b) for a, b in zip(tensors, before))
        scale = min(1.0, factor)
        for t, o in zip(tensors, out):
            if factor > 1:
                assert torch.equal(o, t)
            else:
                u, uw = plain.half_step(t.dtype), plain.half_step(plain.wide_of(t.dtype))
                plain.agrees(o, (scale * plain.f64(t), (u + 3 * uw + 2e-12) * scale * plain.f64(t).abs() + plain.smallest(t.dtype)), "clipped")
    assert torch.equal(layers.clip_by_global_norm(tensors, 0.37 * want), norm)
    inplace = [torch.empty_like(t) for t in before]
    layers.clip_by_global_norm(before, 0.37 * want, out=inplace)
    assert all(torch.equal(a, b) for a, b in zip(tensors, inplace))


def test_global_norm_of_trees_and_layouts(layers):
    a, b, c = normal((6, 5), torch.float64, 1), normal((4, 3, 2), torch.float32, 2), normal((7,), torch.bfloat16, 3)
    tree = {"params": {"z": a, "b": [b, c]}}
    want = math.sqrt(sum(float((t.double() ** 2).sum()) for t in (a, b, c)))
    assert abs(float(layers.global_norm(tree)) - want) < 1e-13 * want
    assert abs(float(layers.global_norm([a.t(), b.permute(2, 0, 1), c])) - want) < 1e-13 * want
    out = {"params": {"b": [torch.empty_like(b), torch.empty_like(c)], "z": torch.empty_like(a)}}      # (another insertion order)
    layers.clip_by_global_norm(tree, 0.5 * want, out=out)
    assert torch.allclose(out["params"]["z"], 0.5 * a, rtol=1e-13, atol=0)
    assert abs(float(layers.global_norm([a, a])) - math.sqrt(2) * float(torch.linalg.norm(a))) < 1e-12
    for call in (lambda: layers.global_norm(a[:, :3]), lambda: layers.global_norm(a[0].expand(3, 5)), lambda: layers.clip_by_global_norm([a, b], 1.0, out=[a]),
                 lambda: layers.clip_by_global_norm(a, 1.0, out=a.t()), lambda: layers.clip_by_global_norm(a, 1.0, out=torch.empty(6, 5, device="cuda")),
                 lambda: layers.global_norm([a, a.cpu()])):
        with pytest.raises(ValueError):
            call()
    from vmc_pde_amd import _native as nat
    for tensors in ([a, a], [a.view(-1)[:20], a.view(-1)[19:]]):
        with pytest.raises(nat.VmcpdeError, match="overlaps"):
            layers.clip_by_global_norm(tensors, 1.0)


def test_clipping_nothing(layers):
    for tensors in ([torch.empty(0, device="cuda")], [torch.empty((3, 0), device="cuda", dtype=torch.bfloat16)] * 200):
        assert float(layers.global_norm(tensors)) == 0 and float(layers.clip_by_global_norm(tensors, 0.0)) == 0


def test_both_readers_of_a_list_of_tensors(layers, monkeypatch):
    """The native form and the Python code that it spares the host from: the same results, the same refusals."""
    from vmc_pde_amd import _native as nat
    assert nat.layer_calls() is not None
    tensors = parts([7, 0, 300, 41, 1], DTYPES, 3)
    out = [torch.empty_like(t) for t in tensors]
    nested = [tensors[0], [tensors[1], (tensors[2],)], {"a": tensors[3], "b": tensors[4]}]
    first = layers.clip_by_global_norm(tensors, 0.1, out=out)
    kept = [o.clone() for o in out]
    assert torch.equal(layers.global_norm(nested), first) and torch.equal(layers.clip_by_global_norm(tuple(tensors), 0.1, out=tuple(out)), first)
    bad = [(tensors, out[:-1]), (tensors, out[::-1]), ([tensors[0]], [out[0][:-1]]), ([tensors[0]], [out[0].cpu()]), ([tensors[0].cpu()], None)]
    parameter = torch.nn.Parameter(tensors[2].clone())
    for native in (True, False):
        if not native:
            monkeypatch.setattr(nat, "_calls", (None,))
        again = layers.clip_by_global_norm(tensors, 0.1, out=out)
        assert torch.equal(again, first) and all(torch.equal(a, b) for a, b in zip(out, kept))
        for t, o in bad:
            with pytest.raises(ValueError):
                layers.clip_by_global_norm(t, 0.1, out=o)
        with pytest.raises(TypeError):
            layers.global_norm([tensors[0], tensors[0].int()])
        with pytest.raises(ValueError, match="no_grad"):
            layers.clip_by_global_norm([parameter], 0.1)
        assert float(layers.global_norm([parameter])) > 0
        with torch.no_grad():
            layers.clip_by_global_norm([parameter], 0.1)
        for empty in ([], [[]], {}):
            with pytest.raises(ValueError, match="no tensors"):
                layers.global_norm(empty)


def test_global_norm_of_extreme_numbers(layers):
    def norm(*v, dtype=torch.float64):
        return float(layers.global_norm(torch.tensor(v, dtype=dtype, device="cuda")))
    assert abs(norm(3e300, 4e300) / 5e300 - 1) < 1e-15 and abs(norm(3e-300, 4e-300) / 5e-300 - 1) < 1e-15 and norm(5e-324) == 5e-324
    assert abs(norm(3e200, 4e200, 1.0, 1e-300) / 5e200 - 1) < 1e-15 and norm(0.0, 0.0) == 0 and norm(1.0, 1e-200) == 1
    assert abs(norm(3e38, 3e38, dtype=torch.float32) / (float(torch.tensor(3e38)) * math.sqrt(2)) - 1) < 1e-14
    assert norm(1e-45, dtype=torch.float32) == float(torch.tensor(1e-45))
    assert norm(math.inf, 1.0) == math.inf and math.isnan(norm(math.nan, math.inf)) and norm(1.0, math.inf, dtype=torch.bfloat16) == math.inf
    for n in (40, 50000):                       # both launches
        t = torch.ones(n, device="cuda")
        t[3] = math.nan
        assert math.isnan(float(layers.clip_by_global_norm(t, 1.0))) and float(t[4]) == 1
        t[3] = math.inf
        assert float(layers.clip_by_global_norm(t, 1.0)) == math.inf and float(t[4]) == 0 and math.isnan(float(t[3]))
        t = torch.ones(n, device="cuda")
        layers.clip_by_global_norm(t, 0.0)
        assert not bool(t.any())
        layers.clip_by_global_norm(t, 0.0)
        assert not bool(t.any())
        t = torch.full((n,), 3.0, device="cuda")
        layers.clip_by_global_norm(t, math.inf)
        assert bool((t == 3).all())


def test_global_norm_beyond_32_bits(layers):
    t = torch.ones((1 << 32) + 4097, dtype=torch.float16, device="cuda")
    norm = layers.clip_by_global_norm(t, 2.0 ** 15)
    assert abs(float(norm) / math.sqrt((1 << 32) + 4097) - 1) < 1e-12
    want = torch.tensor(2.0 ** 15 / float(norm), dtype=torch.float32).half()
    assert float(t[0]) == float(want) and float(t[-1]) == float(want) and bool((t[-5000:] == want.cuda()).all())


# ---- together ----------------------------------------------------------------------------------------------------------------------------

class Block:
    """x + W2 act(W1 norm(x) + b1) + b2 with the squared distance to a target as its loss: the operators as a training step uses them."""

    def __init__(self, dim, hidden, dtype, seed):
        self.names = ["norm_weight", "norm_bias", "w1", "b1", "w2", "b2"]
        shapes = [(dim,), (dim,), (dim, hidden), (hidden,), (hidden, dim), (dim,)]
        self.flat = torch.empty(sum(math.prod(s) for s in shapes), dtype=dtype, device="cuda")    # leaves as views of one vector, as VarState's
        self.p, at = {}, 0
        for k, (name, shape) in enumerate(zip(self.names, shapes)):
            n = math.prod(shape)
            self.p[name] = self.flat[at:at + n].view(shape)
            self.p[name].copy_(normal(shape, dtype, seed + k, 1.0 if len(shape) == 1 else shape[0] ** -0.5))
            at += n

    def step(self, layers, x, target, rate, max_norm):
        p = self.p
        h, mean, rstd = layers.layer_norm(x, p["norm_weight"], p["norm_bias"], want_stats=True)
        a, slope = layers.dense(h, p["w1"], p["b1"], activation="gelu", want_slope=True)
        y = layers.dense(a, p["w2"], p["b2"], residual=x)
        dy = (y - target) * (2 / y.numel())
        da, dw2, db2 = layers.dense_backward(dy, a, p["w2"])
        dh, dw1, db1 = layers.dense_backward(da, h, p["w1"], slope)
        dx, dnw, dnb = layers.layer_norm_backward(dh, x, mean, rstd, p["norm_weight"])
        dx = dx + dy
        grads = dict(zip(self.names, (dnw, dnb, dw1, db1, dw2, db2)))
        norm = layers.clip_by_global_norm(grads, max_norm)
        for name in self.names:
            p[name].sub_(rate * grads[name])
        return norm, dx, grads

    def plain_step(self, flat, x, target, rate, max_norm):
        """The same in torch's automatic differentiation, in fp64 on the CPU."""
        p, at = {}, 0
        for name in self.names:
            n = self.p[name].numel()
            p[name] = flat[at:at + n].view(self.p[name].shape).clone().requires_grad_()
            at += n
        x = x.clone().requires_grad_()
        h = torch.nn.functional.layer_norm(x, x.shape[-1:], p["norm_weight"], p["norm_bias"], 1e-6)
        y = x + torch.nn.functional.gelu(h @ p["w1"] + p["b1"]) @ p["w2"] + p["b2"]
        loss = ((y - target) ** 2).mean()
        grads = torch.autograd.grad(loss, [p[n] for n in self.names] + [x])
        norm = torch.sqrt(sum((g ** 2).sum() for g in grads[:-1]))
        factor = min(1.0, max_norm / float(norm))
        return norm, grads[-1], torch.cat([(p[n] - rate * factor * g).detach().reshape(-1) for n, g in zip(self.names, grads)])


@pytest.mark.parametrize("dtype, tolerance", [(torch.float64, 1e-12), (torch.float32, 2e-5), (torch.bfloat16, 3e-2)], ids=["f64", "f32", "bf16"])
@pytest.mark.parametrize("dim, hidden", [(40, 96), (21, 77)])
def test_a_training_step(layers, dtype, tolerance, dim, hidden):
    """Six roundings deep (16-bit types round every tensor between the operators, 2^-8 each at most, and dy = y - target once more): 8 x 2^-8 in the 2-norm;
    fp32 and fp64 sums of some hundred terms."""
    block = Block(dim, hidden, dtype, 1)
    x, target = normal((3, 50, dim), dtype, 50), normal((3, 50, dim), dtype, 51)
    flat = block.flat.double().cpu()
    norm, dx, _ = block.step(layers, x, target, 0.5, 0.05)
    want_norm, want_dx, want_flat = block.plain_step(flat, x.double().cpu(), target.double().cpu(), 0.5, 0.05)
    assert abs(float(norm) / float(want_norm) - 1) < tolerance
    assert float(torch.linalg.norm(dx.double().cpu() - want_dx) / torch.linalg.norm(want_dx)) < tolerance
    assert float(torch.linalg.norm(block.flat.double().cpu() - want_flat) / torch.linalg.norm(want_flat)) < tolerance


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_training_step_in_a_graph(layers, dtype):
    """Captured once and replayed, with eager work and synchronisations between: each replay is the eager step bit for bit."""
    eager, captured = Block(40, 200, dtype, 1), Block(40, 200, dtype, 1)
    x, target = normal((70, 40), dtype, 50), normal((70, 40), dtype, 51)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step(layers, x, target, 0.1, 0.05)
    torch.cuda.current_stream().wait_stream(side)
    captured.flat.copy_(eager.flat)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, dx, _ = captured.step(layers, x, target, 0.1, 0.05)
    for _ in range(4):
        graph.replay()
        want = eager.step(layers, x, target, 0.1, 0.05)
        torch.cuda.synchronize()
        assert torch.equal(norm, want[0]) and torch.equal(dx, want[1]) and torch.equal(captured.flat, eager.flat)
        x.copy_(normal(x.shape, dtype, 60))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [1, 3, 20])
def test_a_token_in_a_graph(layers, dtype, rows):
    """A block's forward pass for single tokens and a small set clipped, captured and replayed with eager work between: the eager results bit for bit."""
    x = normal((rows, 512), dtype, 1)
    up, down = normal((512, 700), dtype, 2, 0.05), normal((512, 700), dtype, 3, 0.05).t()
    weight, small = normal((512,), dtype, 4), [normal((n,), dtype, 5 + n) for n in (1, 70, 513)]

    def token():
        h = layers.dense(layers.layer_norm(x, weight), up, activation="silu")
        y = layers.dense(h, down, residual=x)
        out = [torch.empty_like(v) for v in small]
        return (y, layers.clip_by_global_norm(small, 0.5, out=out), *out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token()
    for k in range(4):
        graph.replay()
        want = token()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        x.copy_(normal(x.shape, dtype, 60 + k))


def test_two_threads_at_once(layers):
    """Python threads on streams of their own (a call releases the interpreter while it launches)."""
    import threading
    x = [normal((1 + k, 600), torch.bfloat16, k) for k in range(4)]
    kernel = normal((600, 900), torch.bfloat16, 9, 0.05)
    want = [layers.dense(v, kernel, activation="gelu") for v in x]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
            results = [layers.dense(x[k], kernel, activation="gelu") for _ in range(50)]
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(r, want[k]) for r in results):
                wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_streams_at_once(layers):
    """The same operators on two streams: neither disturbs the other (every call has its own workspace)."""
    x = [normal((3000, 200), torch.float32, k) for k in range(2)]
    kernel = [normal((200, 30), torch.float32, 10 + k) for k in range(2)]
    dy = [normal((3000, 30), torch.float32, 20 + k) for k in range(2)]
    want = [layers.dense_backward(dy[k], x[k], kernel[k], scale=3.0) + (layers.global_norm([x[k], dy[k]]),) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(layers.dense_backward(dy[k], x[k], kernel[k], scale=3.0) + (layers.global_norm([x[k], dy[k]]),))
    torch.cuda.synchronize()
    for k in range(2):
        for result in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[k]))


def test_the_flow_from_its_dense_layers(layers):
    """The coupling flow's log density rebuilt from dense operators on the leaves of the parameter vector (net.py:53-61, 95-118) is what the flow kernels
    compute: 32 layers of 21 terms in fp64."""
    from helpers_product import build_varstate
    dim, depth, hidden, n = 2, 4, (21, 21), 500
    ups, downs = [[k % 2] for k in range(depth)], [[1 - k % 2] for k in range(depth)]
    probe = build_varstate(dim, depth, hidden, "Gauss", "no_add", [0.0, 0.0], ups, downs, torch.zeros(4213, dtype=torch.float64))
    theta = probe.net.init(3, out_scale=0.05, hidden_scale=0.5)
    probe.set_parameters(theta)
    x = normal((n, dim), torch.float64, 5)
    blocks, state, log_jac = probe.params["params"]["myINN"], x.clone(), torch.zeros(n, dtype=torch.float64, device="cuda")

    def conditioner(net, u):
        for k in range(3):
            leaf = net[f"Dense_{k}"]
            u = layers.dense(u, leaf["kernel"], leaf["bias"], activation="tanh", scale=10.0 if k == 2 else 1.0)
        return u
    for b in range(depth):
        up, down = state[:, ups[b]], state[:, downs[b]]
        s2 = conditioner(blocks[f"blocks_{b}"]["s2"], down)
        up = up * torch.exp(s2)
        s1 = conditioner(blocks[f"blocks_{b}"]["s1"], up)
        down = down * torch.exp(s1)
        state[:, ups[b]], state[:, downs[b]] = up, down
        log_jac += s1.sum(1) + s2.sum(1)
    logp = -0.5 * (state ** 2).sum(1) - math.log(2 * math.pi) + log_jac
    assert float((logp - probe(x[None], mode="eval")[0]).abs().max()) < 1e-11 * float(logp.abs().max())


def test_clipped_likelihood_gradient(layers):
    """VarState's likelihood gradient (var_state.py:45-53), clipped."""
    import vmc_pde_amd as V
    vs = V.VarState(V.Sampler(key=1, dim=2, name="Gauss", mcmc_info={"offset": [0.0, 0.0], "bound": 0.25}), 2, 1, 2,
                    network_args={"intmediate": (5,), "offset": [0.0, 0.0], "latentSpaceName": "Gauss", "dim": 2})
    x = normal((1, 300, 2), torch.float64, 1, 2.0)
    value, grad = vs(x, mode="costfun", avg=True)
    size = float(torch.linalg.norm(grad))
    clipped_value, clipped = vs(x, mode="costfun", avg=True, max_norm=0.25 * size)
    assert torch.equal(value, clipped_value) and torch.allclose(clipped, 0.25 * grad, rtol=1e-12, atol=0)
    assert torch.equal(vs(x, mode="costfun", avg=True, max_norm=4 * size)[1], grad)
    for bad in (dict(mode="costfun"), dict(mode="eval", avg=True)):
        with pytest.raises(ValueError, match="max_norm"):
            vs(x, max_norm=1.0, **bad)
