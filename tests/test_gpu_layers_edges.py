"""The layer operators at the edges of their types' ranges, of torch's bookkeeping and of what their layouts allow."""
import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import helpers_layers as plain
from test_gpu_layers import DTYPES, IDS, layers, normal  # noqa: F401  (layers: the fixture)

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]
HALF_IDS = ["f16", "bf16"]


@pytest.fixture(params=[True, False], ids=["native", "python"])
def either(request, monkeypatch):
    """Both forms of a call: the native module, and the Python code that it spares the host from."""
    from vmc_pde_amd import _native as nat
    if not request.param:
        monkeypatch.setattr(nat, "_calls", (None,))


# ---- dense -------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("with_slope", [True, False], ids=["slope", "no-slope"])
@pytest.mark.parametrize("dtype", HALF, ids=HALF_IDS)
@pytest.mark.parametrize("size", [(2, 24, 40), (70, 24, 40), (3000, 33, 51), (5, 2000, 300), (600, 300, 520)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("scale, dy_size, operand_size", [(10.0, 7000.0, 1e-3), (1e-4, 1e-3, 30.0)], ids=["large", "small"])
def test_dense_backward_keeps_the_range_of_dy(layers, scale, dy_size, operand_size, size, dtype, with_slope):  # noqa: F811
    """Gradients that fit their type where scale * dy itself does not: beyond fp16's largest number, or among its subnormal ones.  In the 2-norm: one rounding of
    slope * dy and one of the output, at most a half step each, and fp32 sums that cost less than a third one."""
    rows, n_in, n_out = size
    x, kernel = normal((rows, n_in), dtype, 1, operand_size), normal((n_in, n_out), dtype, 2, operand_size)
    dy = normal((rows, n_out), dtype, 3).clamp(-1.5, 1.5) * dy_size
    kept = layers.SLOPE[dtype]
    slope = (0.5 + 0.5 * torch.rand((rows, n_out), generator=torch.Generator().manual_seed(4))).to(kept).cuda() if with_slope else None
    dx, dkernel, _ = layers.dense_backward(dy, x, kernel, slope, scale=scale, want_bias=False)
    dz = scale * plain.f64(dy) * (plain.f64(slope) if with_slope else 1)
    for name, got, want in (("dx", dx, dz @ plain.f64(kernel).t()), ("dkernel", dkernel, plain.f64(x).t() @ dz)):
        assert bool(torch.isfinite(got).all()), f"{name}: not finite"
        # the smallest gradients (2 rows, small: dkernel of some 4e-6) are among fp16's subnormal numbers: there the output's own rounding costs half of its fixed
        # step, 2^-25 = 3e-8, an element, root (elements) times that in the 2-norm
        off, size_ = float(torch.linalg.norm(plain.f64(got) - want)), float(torch.linalg.norm(want))
        assert off <= 3 * plain.half_step(dtype) * size_ + math.sqrt(want.numel()) * plain.smallest(dtype), f"{name}: off by {off / size_:.3g}"


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16], ids=["f64", "bf16"])
def test_dense_copies_rows_that_lie_too_far_apart(layers, dtype):  # noqa: F811
    """Row pitches beyond the kernels' 2^22 (2^21 in fp64) elements."""
    pitch = (1 << 22) + 6
    whole = torch.zeros((60, pitch), dtype=dtype, device="cuda")
    for rows, n_in, n_out in ((3, 60, 50), (7, 50, 60)):
        x, kernel, dy = whole[:rows, 10:10 + n_in], whole[:n_in, 200:200 + n_out], whole[:rows, 400:400 + n_out]
        for k, t in enumerate((x, kernel, dy)):
            t.copy_(normal(t.shape, dtype, k))
        apart = whole[:n_out, 600:600 + n_in]
        apart.copy_(kernel.t())
        for far in (kernel, apart.t()):
            y, slope = layers.dense(x, far, activation="tanh", want_slope=True)
            clean = layers.dense(x.clone(), kernel.clone(), activation="tanh", want_slope=True)
            want = plain.dense(x, kernel, None, None, "tanh", 1.0, dy, dtype)
            plain.agrees(y, want["y"], "y")
            assert torch.equal(slope, clean[1]) or far is not kernel
            for name, got in zip(("dx", "dkernel", "dbias"), layers.dense_backward(dy, x, far, slope)):
                plain.agrees(got, want[name], name)


# ---- layer norm --------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cols", [9, 21, 33, 129, 257, 500, 1025])
def test_layer_norm_of_equal_elements_is_equal(layers, dtype, cols):  # noqa: F811
    """Every lane of a row has the row's sums to the last bit: what is equal in x (and dy) is equal in y (and dx), wherever it stands in the row."""
    rows, g = 600, torch.Generator().manual_seed(cols)
    which = torch.randint(0, 4, (rows, cols), generator=g)
    x, dy = (torch.randn((rows, 4), generator=g, dtype=torch.float64).to(dtype).gather(1, which).cuda() for _ in range(2))
    y, mean, rstd = layers.layer_norm(x, want_stats=True)
    dx, _, _ = layers.layer_norm_backward(dy, x, mean, rstd)
    for name, t in (("y", y), ("dx", dx)):
        for v in range(4):
            mine = (which == v).cuda()
            low, high = t.masked_fill(~mine, math.inf).amin(1), t.masked_fill(~mine, -math.inf).amax(1)
            there = mine.any(1)
            assert torch.equal(low[there], high[there]), name


@pytest.mark.parametrize("offset", [1e3, 1e4, 1e5])
@pytest.mark.parametrize("cols", [3, 21, 100, 1000, 1024, 5000, 20001])
def test_layer_norm_of_rows_far_from_zero(layers, cols, offset):  # noqa: F811
    """fp32 rows of unit spread.  With u = 2^-24 and sums of depth D: the deviations from a first mean are rounded once (u) whatever that mean's own error; what it is
    off by, the deviations' mean, is found to D u of their size and taken off (u); the variance is off by twice that and (D + 4) u, 1 / sqrt by half of it
    and 6 u; two more roundings to y.  In all (|y| + 1) (3 D + 16) u, whatever the offset."""
    x = (normal((40, cols), torch.float64, cols) + offset * (1 + 0.1 * normal((40, 1), torch.float64, cols + 1))).float()
    y, mean, rstd = layers.layer_norm(x, eps=1e-6, want_stats=True)
    exact = plain.f64(x)
    centre = exact.mean(1, keepdim=True)
    want_rstd = 1 / torch.sqrt(((exact - centre) ** 2).mean(1, keepdim=True) + 1e-6)
    want, u, depth = (exact - centre) * want_rstd, 2.0 ** -24, 80 + cols / 512
    plain.agrees(y, (want, (want.abs() + 1) * (3 * depth + 16) * u), "y")
    plain.agrees(rstd, (want_rstd[:, 0], want_rstd[:, 0] * (2 * depth + 12) * u), "rstd")
    # the mean: the nearest fp32 number, but for the correction's own error
    plain.agrees(mean, (centre[:, 0], 1.01 * u * centre[:, 0].abs() + (depth + 4) * u * (exact - centre).abs().mean(1)), "mean")


@pytest.mark.parametrize("dtype", HALF, ids=HALF_IDS)
@pytest.mark.parametrize("cols, spread", [(7, 1.0), (100, 1.0), (1000, 1.0), (8192, 1.0), (8192, 20.0), (40000, 1.0)])
def test_layer_norm_of_16_bit_rows_far_from_zero(layers, dtype, cols, spread):  # noqa: F811
    """Numbers around 300, in steps of 1/4 (fp16) and 2 (bf16).  As above, but with the first mean as it is, which is off by its own last place and one of a sum that is
    exact up to 2^13 and 2^16 numbers (beyond, D / 80 more): 4 u |mean| / standard deviation on every y; and the output's rounding."""
    x = (300 + spread * normal((40, cols), torch.float64, cols)).to(dtype)
    y, mean, rstd = layers.layer_norm(x, eps=1e-6, want_stats=True)
    exact = plain.f64(x)
    centre = exact.mean(1, keepdim=True)
    want_rstd = 1 / torch.sqrt(((exact - centre) ** 2).mean(1, keepdim=True) + 1e-6)
    want, u, depth = (exact - centre) * want_rstd, 2.0 ** -24, 80 + cols / 512
    bound = (want.abs() + 1) * ((3 * depth + 16) * u + 4 * depth / 80 * u * centre.abs() * want_rstd)
    plain.agrees(y, (want, bound + plain.half_step(dtype) * (want.abs() + bound) + plain.smallest(dtype)), "y")


# ---- global norm -------------------------------------------------------------------------------------------------------------------------

def test_global_norm_of_many_large_numbers(layers):  # noqa: F811
    """More than 2^24 numbers just below 2^500, whose squares add up to more than the largest fp64 number while their norm is some 2^512; and as many tiny ones."""
    n = 18500000
    for value in (0.99 * 2.0 ** 500, 0.99 * 2.0 ** 470, 1.01 * 2.0 ** -500):
        t = torch.full((n,), value, dtype=torch.float64, device="cuda")
        want = math.sqrt(n) * value
        assert abs(float(layers.global_norm(t)) / want - 1) < 1e-12      # (some thousand additions of positive numbers in a row, 2^-53 each)
        norm = layers.clip_by_global_norm(t, 1.0)
        assert abs(float(norm) / want - 1) < 1e-12
        if want > 1:
            assert abs(float(t[0]) * math.sqrt(n) - 1) < 1e-12 and bool((t == t[0]).all())


@pytest.mark.parametrize("dtype, size, max_norm", [(torch.float32, 1e37, 1e-3), (torch.float32, 1e37, 1e-28), (torch.bfloat16, 1e37, 1e-3), (torch.bfloat16, 1e37, 1e-28),
                                                   (torch.float64, 1e300, 1e-15), (torch.float64, 1e300, 1e-280), (torch.float64, 1e-150, 1e-290)],
                         ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("sizes", [[40], [300, 7, 21], [9000, 2000], [50000, 300], [300] * 130], ids=["40", "leaves", "9000", "50000", "130"])
@pytest.mark.parametrize("mixed", [False, True], ids=["one-type", "mixed"])
def test_clipping_far(layers, dtype, size, max_norm, sizes, mixed):  # noqa: F811
    """max_norm / norm below the smallest normal number of the arithmetic: the clipped elements, which are ordinary numbers, keep their digits."""
    tensors = [normal((n,), dtype, k, size) for k, n in enumerate(sizes)] + ([torch.ones(5, device="cuda", dtype=torch.float32)] if mixed else [])
    exact = [plain.f64(t) for t in tensors]
    largest = max(float(t.abs().max()) for t in exact)
    norm = largest * math.sqrt(math.fsum(float(((t / largest) ** 2).sum()) for t in exact))
    got = layers.clip_by_global_norm(tensors, max_norm)
    assert abs(float(got) / norm - 1) < 1e-12
    for t, e in zip(tensors, exact):
        want = e / norm * max_norm if max_norm > 1e-200 else (e / norm) * max_norm
        u, uw = plain.half_step(t.dtype), plain.half_step(plain.wide_of(t.dtype))
        plain.agrees(t, (want, (u + 3 * uw + 2e-12) * want.abs() + 1.01 * plain.smallest(t.dtype)), "clipped")


# ---- errors, and what torch keeps account of -----------------------------------------------------------------------------------------------

def test_a_call_that_failed_after_its_launch_is_not_made_again(layers):  # noqa: F811
    """rc -1 is a refusal before any launch, which the Python code calls again and reports; any other error is raised as it is, with nothing run twice."""
    from vmc_pde_amd import _native as nat
    calls, library = nat.layer_calls(), nat.lib()
    t, x, kernel = torch.full((10,), 2.0, device="cuda"), normal((3, 4), torch.float32, 1), normal((4, 5), torch.float32, 2)
    y, mean, rstd = layers.layer_norm(x, want_stats=True)
    names = ("vmcpde_dense_workspace_bytes", "vmcpde_dense", "vmcpde_dense_backward", "vmcpde_layer_norm", "vmcpde_layer_norm_backward_workspace_bytes",
             "vmcpde_layer_norm_backward", "vmcpde_global_norm_workspace_bytes", "vmcpde_global_norm")      # (the order that bind takes them in)
    seen = []

    def entry(name, result):
        """What stands for an entry point: needs no workspace, launches nothing, returns `result`."""
        restype, argtypes = nat._PROTOS[name]

        def stand_in(*arguments):
            seen.append(name)
            return 0 if name.endswith("_bytes") else result
        return C.CFUNCTYPE(restype, *[a if a in (C.c_int32, C.c_int64, C.c_double) else C.c_void_p for a in argtypes])(stand_in)

    every = {"vmcpde_dense": lambda: layers.dense(x, kernel), "vmcpde_dense_backward": lambda: layers.dense_backward(normal((3, 5), torch.float32, 3), x, kernel),
             "vmcpde_layer_norm": lambda: layers.layer_norm(x), "vmcpde_layer_norm_backward": lambda: layers.layer_norm_backward(y, x, mean, rstd),
             "vmcpde_global_norm": lambda: layers.clip_by_global_norm([t], 1.0)}
    for result in (-2, -1):
        stand_ins = [entry(name, result) for name in names]
        calls.bind(*(C.cast(f, C.c_void_p).value for f in stand_ins))
        try:
            for name, call in every.items():
                seen.clear()
                if result == -2:
                    with pytest.raises(nat.VmcpdeError, match=name):
                        call()
                else:
                    call()                                   # (refused here, done by the Python code through the library's own entry)
                assert seen.count(name) == 1
            if result == -2:
                assert bool((t == 2).all())
        finally:
            calls.bind(*(C.cast(getattr(library, name), C.c_void_p).value for name in names))
    assert float(layers.global_norm([t])) == pytest.approx(1.0, rel=1e-6)


def test_clipping_in_place_is_seen_by_automatic_differentiation(layers, either):  # noqa: F811
    for own in (True, False):
        saved, given = torch.full((8,), 3.0, device="cuda"), torch.full((8,), 3.0, device="cuda")
        x = torch.ones(8, device="cuda", requires_grad=True)
        loss = (x * saved).sum()
        before = saved._version
        assert float(layers.global_norm([saved])) > 1 and saved._version == before
        with torch.no_grad():
            layers.clip_by_global_norm([saved] if own else [given], 1.0, out=None if own else [saved])
        assert given._version == 0
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        free = torch.full((8,), 3.0, device="cuda")
    layers.clip_by_global_norm([free], 1.0)                  # (such tensors have no account to keep)
    assert float(layers.global_norm([free])) == pytest.approx(1.0, rel=1e-6)


def test_forward_mode_tangents_are_refused(layers, either):  # noqa: F811
    x, kernel, bias, dy = normal((3, 4), torch.float32, 1), normal((4, 5), torch.float32, 2), normal((5,), torch.float32, 3), normal((3, 5), torch.float32, 4)
    weight, slope = normal((4,), torch.float32, 5), torch.ones((3, 5), device="cuda")
    y, mean, rstd = layers.layer_norm(x, want_stats=True)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: layers.dense(dual(x), kernel), lambda: layers.dense(x, dual(kernel)), lambda: layers.dense(x, kernel, dual(bias)),
                     lambda: layers.dense(x, kernel, residual=dual(dy)), lambda: layers.dense_backward(dual(dy), x, kernel), lambda: layers.dense_backward(dy, dual(x), kernel),
                     lambda: layers.dense_backward(dy, x, dual(kernel)), lambda: layers.dense_backward(dy, x, kernel, dual(slope)), lambda: layers.layer_norm(dual(x)),
                     lambda: layers.layer_norm(x, dual(weight)), lambda: layers.layer_norm(x, weight, dual(weight)), lambda: layers.layer_norm_backward(dual(x), x, mean, rstd),
                     lambda: layers.layer_norm_backward(x, dual(x), mean, rstd), lambda: layers.layer_norm_backward(x, x, dual(mean), rstd),
                     lambda: layers.layer_norm_backward(x, x, mean, dual(rstd)), lambda: layers.layer_norm_backward(x, x, mean, rstd, dual(weight)),
                     lambda: layers.global_norm([x, dual(weight)]), lambda: layers.clip_by_global_norm([dual(weight)], 1.0),
                     lambda: layers.clip_by_global_norm([weight], 1.0, out=[dual(torch.empty_like(weight))])):
            with pytest.raises(ValueError, match="autograd"):
                call()
        assert torch.equal(layers.layer_norm(x), y)          # what has no tangent is taken there too
