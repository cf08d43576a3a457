"""Layer operators of a fit: the dense layer with its epilogue, layer norm, and the global gradient norm.

The conditioners of the coupling flow are chains of dense layers (reference: vmc_fluids/net.py:53-61) that `csrc/flow.hip` evaluates whole,
per sample, with their weights in LDS.  These are the same layers as operators over a batch, of any width, in fp64, fp32, fp16 and bf16, with
what a training step of a wide network needs around them.  Like the rest of this package they are explicit: every operator has its gradient as
a function of its own, and takes no part in torch's automatic differentiation (tensors that require it are refused while it is recording, and so are
those with a forward-mode tangent).

All run on the current HIP stream, allocate through torch, never synchronise with the host, and can be captured into a graph.  Sums, statistics
and epilogues are held in fp32 for fp32 and 16-bit elements, in fp64 for fp64.  None uses atomics: the same call gives the same bits.

Small calls are bound by the host, so each function first hands its arguments to its native form (csrc/layer_calls.cpp), which does the call if
nothing has to be copied or refused.  What follows it here is the whole operator: every layout, and every refusal.
"""
from __future__ import annotations

import ctypes as C
import struct
from array import array

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _native as nat

DTYPE = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
ACTIVATION = {"none": 0, "tanh": 1, "gelu": 2, "silu": 3}
SLOPE = {torch.float64: torch.float64, torch.float32: torch.float32, torch.float16: torch.float32, torch.bfloat16: torch.float16}
WIDE = {torch.float64: torch.float64, torch.float32: torch.float32, torch.float16: torch.float32, torch.bfloat16: torch.float32}
_HALF = (torch.float16, torch.bfloat16)
_AUTOGRAD = "the layer operators are no autograd functions: call them under torch.no_grad() and use their *_backward"
_HOST = "the layer operators run on device (HBM) tensors only"

_pack_dense = struct.Struct("@4i3qPqPqPPqdPqPPqPPP").pack       # vmcpde_dense_args
_pack_norm = struct.Struct("@2i2qPqPPdPqPPPqPPP").pack          # vmcpde_norm_args

_calls, _empty, _recording = nat.layer_calls, torch.empty, torch.is_grad_enabled
# (torch built without a GPU backend lacks these; there every tensor is refused before they are needed)
_device, _stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
_entry = {}


def _entries():
    """The entry points with packed records as their first argument (bound on first use: the library may not be built yet)."""
    library, found = nat.lib(), {}
    for name, (result, arguments) in nat._PROTOS.items():
        if name.startswith(("vmcpde_dense", "vmcpde_layer_norm", "vmcpde_global_norm")):
            f = library[name]
            f.restype, f.argtypes = result, [C.c_void_p, *arguments[1:]]
            found[name] = f
    _entry.update(found)                       # (at once: another thread finds none of them or all)
    return _entry


def _call(name, *arguments):
    rc = (_entry or _entries())[name](*arguments)
    if rc != 0:
        nat.check(rc, name)


def _workspace(name, device, *arguments):
    nbytes = (_entry or _entries())[name](*arguments)
    if nbytes == 0:
        return None, 0
    if nbytes < 0:
        nat.check(-1, name)
    return _empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _plain(t):
    """Refuses what automatic differentiation, in either mode, would follow."""
    if t.requires_grad and _recording() or unpack_dual(t).tangent is not None:
        raise ValueError(_AUTOGRAD)


def _first(t):
    """Element type and device index of the tensor that every other one has to agree with."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"a tensor is needed, not {type(t).__name__}")
    dtype = t.dtype
    if dtype not in DTYPE:
        raise TypeError(f"element type {dtype}: fp64, fp32, fp16 and bf16 are supported")
    _plain(t)
    return dtype, t.get_device()


def _agrees(t, name, dtype, index):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, not {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has type {t.dtype}: {dtype} is needed")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on " + (f"cuda:{index}" if index >= 0 else "cpu"))
    _plain(t)


def _far(dtype):
    """Row pitch from which on the dense kernels, whose offsets within a tile have 31 bits, do not take a matrix."""
    return 1 << (21 if dtype == torch.float64 else 22)


def _rows(t, cols, name, far=None):
    """(tensor, row pitch) of t as a matrix of `cols` columns whose rows' elements lie behind each other, less than `far` apart; copied only where no such
    view exists."""
    if t.dim() == 0 or t.shape[-1] != cols:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: its last axis should have {cols}")
    t = t.resolve_neg()
    if t.is_contiguous():
        return t, cols
    m = t.reshape(-1, cols)
    if cols > 1 and m.stride(1) != 1 or m.shape[0] > 1 and (m.stride(0) < cols or far and m.stride(0) >= far > cols):
        return m.contiguous(), cols
    return m, m.stride(0) if m.shape[0] > 1 else cols


def _same_shape(t, shape, name):
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: {tuple(shape)} is needed")


def _kernel_layout(kernel):
    """(tensor, n_in, n_out, row pitch, whether it is stored (n_out, n_in)) of a kernel of shape (n_in, n_out)."""
    if kernel.dim() != 2:
        raise ValueError(f"kernel has shape {tuple(kernel.shape)}: (n_in, n_out) is needed")
    n_in, n_out = kernel.shape
    if n_in == 0 or n_out == 0:
        raise ValueError(f"kernel has shape {(n_in, n_out)}: no axis may be empty")
    kernel = kernel.resolve_neg()
    (s0, s1), far = kernel.stride(), _far(kernel.dtype)
    if (s1 == 1 or n_out == 1) and (n_out <= s0 < far or n_in == 1):
        return kernel, n_in, n_out, s0 if n_in > 1 else n_out, 0
    if (s0 == 1 or n_in == 1) and (n_in <= s1 < far or n_out == 1):
        return kernel, n_in, n_out, s1 if n_out > 1 else n_in, 1
    return kernel.contiguous(), n_in, n_out, n_out, 0


def dense(x, kernel, bias=None, *, activation="none", scale=1.0, residual=None, want_slope=False):
    """y = scale * act(x @ kernel + bias) + residual, in one pass over x and the kernel.

    x (..., n_in); kernel (n_in, n_out), the layout of the flat parameter vector's leaves, or a transposed view of an (n_out, n_in) one; bias
    (n_out,); residual of y's shape.  activation: "none", "tanh", "gelu" (z Phi(z)), "silu".  `scale` is the output factor of the reference's
    conditioners (net.py:50, 61: 10 * tanh).  Widths are below 2^22 (2^21 in fp64); rows that lie further apart are copied.  With `want_slope` returns (y, slope): act'(z),
    which `dense_backward` takes (None for "none"), of the type SLOPE[x.dtype] (fp16 for bf16, where slopes under 2^-25 become zero; fp32 for fp16, else the element
    type)."""
    calls = _calls()
    if calls is not None:
        device = _device()
        done = calls.dense(x, kernel, bias, ACTIVATION.get(activation, -1), scale, residual, want_slope, device, _stream(device))
        if done is not None:
            return done
    dtype, index = _first(x)
    _agrees(kernel, "kernel", dtype, index)
    if bias is not None:
        _agrees(bias, "bias", dtype, index)
    if residual is not None:
        _agrees(residual, "residual", dtype, index)
    if index < 0:
        raise ValueError(_HOST)
    if _device() != index:
        with torch.cuda.device(index):
            return dense(x, kernel, bias, activation=activation, scale=scale, residual=residual, want_slope=want_slope)
    act = ACTIVATION.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r}: one of {sorted(ACTIVATION)} is needed")
    kernel, n_in, n_out, ldk, kernel_t = _kernel_layout(kernel)
    shape, device = (*x.shape[:-1], n_out), x.device
    x, ldx = _rows(x, n_in, "x", _far(dtype))
    if bias is not None:
        _same_shape(bias, (n_out,), "bias")
        bias = bias.resolve_neg().contiguous()
    ldr = 0
    if residual is not None:
        _same_shape(residual, shape, "residual")
        residual, ldr = _rows(residual, n_out, "residual")
    y = x.new_empty(shape)
    slope = _empty(shape, dtype=SLOPE[dtype], device=index) if want_slope and act else None
    record = _pack_dense(DTYPE[dtype], act, kernel_t, 0, x.numel() // n_in, n_in, n_out, x.data_ptr(), ldx, kernel.data_ptr(), ldk,
                         0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(), ldr, float(scale), y.data_ptr(), n_out,
                         0 if slope is None else slope.data_ptr(), 0, 0, 0, 0, 0)
    ws, nbytes = _workspace("vmcpde_dense_workspace_bytes", device, record, 0)
    _call("vmcpde_dense", record, None if ws is None else ws.data_ptr(), nbytes, _stream(index))
    return (y, slope) if want_slope else y


def dense_backward(dy, x, kernel, slope=None, *, scale=1.0, want_x=True, want_kernel=True, want_bias=True):
    """(dx, dkernel, dbias) of `dense` for the gradient dy of y, None where not wanted: with dz = scale * slope * dy, dx = dz @ kernel^T,
    dkernel = x^T @ dz (n_in, n_out), dbias = the sum of dz over the rows.  `slope` and `scale` as the forward call had them; the residual's
    gradient is dy itself.  slope * dy is rounded to the element type, in which the matrix pipe takes it (fp16: it has to stay below 65504, and slopes
    reach 1.13); the scale is applied to the fp32 sums, and dbias sums unrounded numbers.  Tensors cast to fp32 beforehand round nothing on the way."""
    calls = _calls()
    if calls is not None:
        device = _device()
        done = calls.dense_backward(dy, x, kernel, slope, scale, want_x, want_kernel, want_bias, device, _stream(device))
        if done is not None:
            return done
    dtype, index = _first(dy)
    _agrees(x, "x", dtype, index)
    _agrees(kernel, "kernel", dtype, index)
    if index < 0:
        raise ValueError(_HOST)
    if _device() != index:
        with torch.cuda.device(index):
            return dense_backward(dy, x, kernel, slope, scale=scale, want_x=want_x, want_kernel=want_kernel, want_bias=want_bias)
    kernel, n_in, n_out, ldk, kernel_t = _kernel_layout(kernel)
    x_shape, device = x.shape, x.device
    shape = (*x_shape[:-1], n_out)
    _same_shape(dy, shape, "dy")
    x, ldx = _rows(x, n_in, "x", _far(dtype))
    dy, ldd = _rows(dy, n_out, "dy", _far(dtype))
    if slope is not None:
        _agrees(slope, "slope", SLOPE[dtype], index)
        _same_shape(slope, shape, "slope")
        slope = slope.resolve_neg().contiguous()
    dx = x.new_empty(x_shape) if want_x else None
    dkernel = x.new_empty((n_in, n_out)) if want_kernel else None
    dbias = x.new_empty(n_out) if want_bias else None
    record = _pack_dense(DTYPE[dtype], 0, kernel_t, 0, x.numel() // n_in, n_in, n_out, x.data_ptr(), ldx, kernel.data_ptr(), ldk, 0, 0, 0, float(scale), 0, 0,
                         0 if slope is None else slope.data_ptr(), dy.data_ptr(), ldd, 0 if dx is None else dx.data_ptr(),
                         0 if dkernel is None else dkernel.data_ptr(), 0 if dbias is None else dbias.data_ptr())
    ws, nbytes = _workspace("vmcpde_dense_workspace_bytes", device, record, 1)
    _call("vmcpde_dense_backward", record, None if ws is None else ws.data_ptr(), nbytes, _stream(index))
    return dx, dkernel, dbias


def _weights(t, name, dtype, index, cols):
    """A weight or bias of the layer norm: x's element type, or fp32 beside 16-bit elements."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, not {type(t).__name__}")
    if t.dtype != dtype and not (t.dtype == torch.float32 and dtype in _HALF):
        raise TypeError(f"{name} has type {t.dtype} beside {dtype}: the same, or fp32 beside 16-bit elements")
    _agrees(t, name, t.dtype, index)
    _same_shape(t, (cols,), name)
    return t.resolve_neg().contiguous()


def _columns(x):
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x has shape {tuple(x.shape)}: a last axis of one or more is needed")
    return x.shape[-1]


def layer_norm(x, weight=None, bias=None, *, eps=1e-6, want_stats=False):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis (the variance is the mean of the squared deviations).

    weight, bias (cols,): x's element type, or fp32 beside 16-bit elements.  With `want_stats` returns (y, mean, rstd), which
    `layer_norm_backward` takes: of the leading shape, fp32 (fp64 for fp64)."""
    calls = _calls()
    if calls is not None:
        device = _device()
        done = calls.layer_norm(x, weight, bias, eps, want_stats, device, _stream(device))
        if done is not None:
            return done
    dtype, index = _first(x)
    cols = _columns(x)
    weights = None
    if weight is not None:
        weight = _weights(weight, "weight", dtype, index, cols)
        weights = weight.dtype
    if bias is not None:
        bias = _weights(bias, "bias", dtype, index, cols)
        if weights is not None and bias.dtype != weights:
            raise TypeError(f"weight has type {weights} and bias {bias.dtype}")
        weights = bias.dtype
    if not eps >= 0:
        raise ValueError(f"eps = {eps}")
    if index < 0:
        raise ValueError(_HOST)
    if _device() != index:
        with torch.cuda.device(index):
            return layer_norm(x, weight, bias, eps=eps, want_stats=want_stats)
    shape, device = x.shape, x.device
    x, ldx = _rows(x, cols, "x")
    y = x.new_empty(shape)
    mean = rstd = None
    if want_stats:
        mean, rstd = _empty((2, *shape[:-1]), dtype=WIDE[dtype], device=index).unbind(0)
    _call("vmcpde_layer_norm", _pack_norm(DTYPE[dtype], DTYPE[weights or dtype], x.numel() // cols, cols, x.data_ptr(), ldx, 0 if weight is None else weight.data_ptr(),
                                          0 if bias is None else bias.data_ptr(), float(eps), y.data_ptr(), cols, 0 if mean is None else mean.data_ptr(),
                                          0 if rstd is None else rstd.data_ptr(), 0, 0, 0, 0, 0), _stream(index))
    return (y, mean, rstd) if want_stats else y


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, want_x=True, want_weight=True, want_bias=True, weight_dtype=None):
    """(dx, dweight, dbias) of `layer_norm` for the gradient dy of y, None where not wanted; mean, rstd from `layer_norm(..., want_stats=True)`,
    where the mean is rounded to fp32 (fp64 for fp64): normalised elements are off by up to 2^-24 |mean| rstd here, though y is not.
    dweight and dbias have the weight's type (without a weight `weight_dtype`, else x's)."""
    calls = _calls()
    if calls is not None and (weight is not None or weight_dtype is None):
        device = _device()
        done = calls.layer_norm_backward(dy, x, mean, rstd, weight, want_x, want_weight, want_bias, device, _stream(device))
        if done is not None:
            return done
    dtype, index = _first(dy)
    _agrees(x, "x", dtype, index)
    cols = _columns(x)
    weights = dtype
    if weight is not None:
        weight = _weights(weight, "weight", dtype, index, cols)
        weights = weight.dtype
    elif weight_dtype is not None:
        if weight_dtype != dtype and not (dtype in _HALF and weight_dtype == torch.float32):
            raise TypeError(f"weight_dtype {weight_dtype} beside {dtype}: the same, or fp32 beside 16-bit elements")
        weights = weight_dtype
    shape, device = x.shape, x.device
    _same_shape(dy, shape, "dy")
    for name, t in (("mean", mean), ("rstd", rstd)):
        _agrees(t, name, WIDE[dtype], index)
        _same_shape(t, shape[:-1], name)
    if index < 0:
        raise ValueError(_HOST)
    if _device() != index:
        with torch.cuda.device(index):
            return layer_norm_backward(dy, x, mean, rstd, weight, want_x=want_x, want_weight=want_weight, want_bias=want_bias, weight_dtype=weight_dtype)
    x, ldx = _rows(x, cols, "x")
    dy, ldd = _rows(dy, cols, "dy")
    mean, rstd = mean.resolve_neg().contiguous(), rstd.resolve_neg().contiguous()
    dx = x.new_empty(shape) if want_x else None
    if want_weight and want_bias:
        dweight, dbias = _empty((2, cols), dtype=weights, device=index).unbind(0)
    else:
        dweight = _empty(cols, dtype=weights, device=index) if want_weight else None
        dbias = _empty(cols, dtype=weights, device=index) if want_bias else None
    record = _pack_norm(DTYPE[dtype], DTYPE[weights], x.numel() // cols, cols, x.data_ptr(), ldx, 0 if weight is None else weight.data_ptr(), 0, 0.0, 0, 0,
                        mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), ldd, 0 if dx is None else dx.data_ptr(), 0 if dweight is None else dweight.data_ptr(),
                        0 if dbias is None else dbias.data_ptr())
    ws, nbytes = _workspace("vmcpde_layer_norm_backward_workspace_bytes", device, record) if want_weight or want_bias else (None, 0)
    _call("vmcpde_layer_norm_backward", record, None if ws is None else ws.data_ptr(), nbytes, _stream(index))
    return dx, dweight, dbias


def _leaves(tree, out):
    if isinstance(tree, torch.Tensor):
        out.append(tree)
    elif isinstance(tree, dict):
        for key in sorted(tree):               # the parameter trees' order, and the same one for a dict and the dict it is written to
            _leaves(tree[key], out)
    elif isinstance(tree, (list, tuple)):
        for v in tree:
            _leaves(v, out)
    else:
        raise TypeError(f"a tensor, or a list or (nested) dict of tensors is needed, not {type(tree).__name__}")
    return out


def _fills_memory(t):
    """Whether t's elements, in whatever order, lie behind each other."""
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _codes(leaves):
    try:
        return [DTYPE[t.dtype] for t in leaves]
    except KeyError as unknown:
        raise TypeError(f"element type {unknown.args[0]}: fp64, fp32, fp16 and bf16 are supported") from None


def _table(leaves, targets, clip):
    """(rows of vmcpde_tensor, device index); refuses what cannot be reduced or written."""
    index, codes = leaves[0].get_device(), _codes(leaves)
    if any([unpack_dual(t).tangent is not None for t in (leaves if targets is None else [*leaves, *targets])]):
        raise ValueError(_AUTOGRAD)
    if index < 0:
        raise ValueError(_HOST)
    if any([t.get_device() != index for t in leaves]):
        raise ValueError(f"tensors on several devices: {sorted({str(t.device) for t in leaves})}")
    plain = all([t.is_contiguous() for t in leaves])
    if not plain:
        for t in leaves:
            if t.numel() and not t.is_contiguous() and not _fills_memory(t):
                raise ValueError(f"a tensor of shape {tuple(t.shape)} and strides {t.stride()} does not fill its memory: pass a contiguous one")
    places = to = [t.data_ptr() for t in leaves]
    if targets is not None:
        if len(targets) != len(leaves):
            raise ValueError(f"{len(leaves)} tensors and {len(targets)} to write them to")
        if [(t.shape, t.is_neg()) for t in targets] != [(t.shape, t.is_neg()) for t in leaves] or _codes(targets) != codes or any([t.get_device() != index for t in targets]) \
                or not (plain and all([t.is_contiguous() for t in targets])) and [t.stride() for t in targets] != [t.stride() for t in leaves]:
            raise ValueError("out: shapes, strides, element types and devices have to be those of the tensors")
        to = [t.data_ptr() for t in targets]
    if clip and _recording() and any([t.requires_grad for t in targets or leaves]):
        raise ValueError("clipping writes into tensors that automatic differentiation records: call it under torch.no_grad()")
    return array("q", [v for row in zip(places, to, [t.numel() for t in leaves], codes) for v in row]), index


def _global_norm(tensors, max_norm, out):
    clip = max_norm is not None
    calls = _calls()
    if calls is not None:
        device = _device()
        done = calls.global_norm(tensors if type(tensors) is list else _leaves(tensors, []), out if out is None or type(out) is list else _leaves(out, []), max_norm,
                                 device, _stream(device))
        if done is not None:
            return done
    leaves = _leaves(tensors, [])
    if not leaves:
        raise ValueError("no tensors")
    table, index = _table(leaves, None if out is None else _leaves(out, []), clip)
    if _device() != index:
        with torch.cuda.device(index):
            return _global_norm(tensors, max_norm, out)
    address, count = table.buffer_info()[0], len(leaves)
    norm = _empty((), dtype=torch.float64, device=index)
    ws, nbytes = _workspace("vmcpde_global_norm_workspace_bytes", index, address, count)
    _call("vmcpde_global_norm", address, count, clip, max_norm if clip else 0.0, norm.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, _stream(index))
    if clip:                                   # written in place: a recorded graph that saved one of these has to see it
        for t in leaves if out is None else _leaves(out, []):
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)
    return norm


def global_norm(tensors):
    """2-norm over all elements of a tensor, or of a list or (nested) dict of them (`VarState.params`), as an fp64 scalar on the device.
    Element types may differ.  Squares are summed in fp64; no finite norm overflows or vanishes on its way."""
    return _global_norm(tensors, None, None)


def clip_by_global_norm(tensors, max_norm, out=None):
    """Multiplies every tensor by max_norm / norm where their `global_norm` exceeds max_norm, in place or into `out` (tensors of the same shapes,
    strides and types), which torch's version counters see.  Returns the norm before clipping; nothing is read back to the host.  A NaN norm leaves the elements as they are, an
    infinite one makes finite elements zero.  Tensors that overlap each other are refused: they would be scaled twice."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm = {max_norm}")
    if out is not None and not isinstance(out, (torch.Tensor, list, tuple, dict)):
        raise TypeError("out: a tensor, or a list or (nested) dict of tensors")
    return _global_norm(tensors, max_norm, out)
